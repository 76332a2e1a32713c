"""Attention over a shared prefix: runs of more pages than a warp knows at a time, caches whose offsets pass 32 bits.  Pages stand in several
tables, which keeps the caches small; the plain form is computed on the device in 64 bits."""
import math
import types

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_shared_prefix import BF16, F32, PAGE, ints, kernels_of, ops, pages_for  # noqa: E402,F401


def call(ops, kv, pool, groups, heads, seed=0):
    """groups: (shared pages, [own cached positions, ...]), a new token a sequence; pool: the page ids that tables are made of."""
    g = torch.Generator().manual_seed(seed)
    kv_heads, dim, dtype = kv.shape[2], kv.shape[4], kv.dtype
    shared, sizes = [p for p, _ in groups], [len(s) for _, s in groups]
    group_of = [i for i, n in enumerate(sizes) for _ in range(n)]
    starts = [PAGE * p + own for p, s in groups for own in s]
    n, width = len(starts), max(pages_for(s + 1) for s in starts)
    deal = lambda k: pool[torch.randint(0, len(pool), (k,), generator=g)].to(torch.int32)      # noqa: E731
    prefix = [deal(p) for p in shared]
    table = torch.stack([torch.cat([prefix[i], deal(width - shared[i])]) for i in group_of])
    q = (torch.randn((n, heads, dim), generator=g) * torch.linspace(0.3, 2.0, heads)[:, None]).to(dtype).cuda()
    lens = [s + 1 for s in starts]
    batch = types.SimpleNamespace(n_seqs=n, n_tokens=n, table_width=width, max_q_len=1, cu_seqlens=ints(list(range(n + 1))), start=ints(starts),
                                  kv_len=ints(lens), page_table=table.cuda(), seq_of_token=ints(list(range(n))), positions=ints(starts), max_kv_len=max(lens))
    scale = 1.0 / math.sqrt(dim)
    got = {}
    launched = kernels_of(ops, lambda: got.update(y=ops.attention_shared(q, kv, batch, ops.SharedPrefix.of(sizes, shared, lens, "cuda"), scale)))
    ops.check_status()
    for b in range(n):
        t = table[b, :pages_for(lens[b])].long().cuda()
        k, v = kv[t].double().permute(1, 2, 0, 3, 4).reshape(2, kv_heads, -1, dim)[:, :, :lens[b]]
        qb = q[b].double().view(kv_heads, -1, dim)
        s = torch.einsum("kgd,kld->kgl", qb, k) * scale
        p = torch.softmax(s, -1)
        want, spread = torch.einsum("kgl,kld->kgd", p, v), torch.einsum("kgl,kld->kgd", p, v.abs())
        # (the bounds of the other tests of this operator: scores, exponential, sums; weights and result in bfloat16)
        off = (torch.einsum("kgd,kld->kgl", qb.abs(), k.abs()) * scale * ((dim + 2) * 2.0 ** -24 + 2.0 ** -22)).amax(-1, keepdim=True)
        rel = 2 * off + 2.0 ** -21 + (lens[b] + 8) * 2.0 ** -23 + (3 * 2.0 ** -9 if dtype == BF16 else 0.0)
        over = ((got["y"][b].double().view_as(want) - want).abs() / (spread * rel + 1e-30)).max().item()
        assert over <= 1.0, f"sequence {b}: an element is off by {over:.3f} times what rounding allows"
    return launched


def cache(pages, kv_heads, dim, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((pages, 2, kv_heads, PAGE, dim), generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("pages,n", [(300, 3), (700, 2), (450, 130)])
def test_runs_of_many_shared_pages(ops, pages, n, dim):
    """Many heads share out the blocks among them: runs of up to some hundred pages, whose numbers are read 32 at a time."""
    kv = cache(60, 64, dim, BF16)
    assert call(ops, kv, torch.arange(1, 60), [(pages, [i * 7 % 90 for i in range(n)])], 64, seed=pages) == 3


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (48, BF16), (64, F32)])
@pytest.mark.parametrize("shared", [0, 1])
def test_runs_of_many_own_pages(ops, shared, dim, dtype):
    kv = cache(40, 64, dim, dtype)
    n = 28 if dtype == BF16 else 6
    assert call(ops, kv, torch.arange(1, 40), [(shared, [2600 + 37 * i for i in range(n)])], 64, seed=dim) == 2


@pytest.mark.parametrize("kv_heads,dim,dtype", [(8, 128, BF16), (8, 64, BF16), (5, 48, BF16), (4, 64, F32)])
def test_offsets_beyond_32_bits(ops, kv_heads, dim, dtype):
    page = 2 * kv_heads * PAGE * dim
    pages = (1 << 31) // page + 200
    kv = torch.empty((pages, 2, kv_heads, PAGE, dim), dtype=dtype, device="cuda")
    kv[-150:] = cache(150, kv_heads, dim, dtype)
    pool = torch.arange(pages - 150, pages)
    for prefix in (3, 400):
        launched = call(ops, kv, pool, [(prefix, [5, 700, 64]), (0, [130])], 4 * kv_heads, seed=prefix)
        assert launched == (3 if prefix == 400 and dim in (64, 128) and dtype == BF16 and 3 * kv_heads * 400 > 3500 * (128 // dim) else 2)
