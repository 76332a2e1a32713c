"""Draws from rows in which tokens are ruled out (-inf): none of them comes, whatever the uniform number."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from wick_b200.sampling.sampler import SamplerConfig, pick_from_sorted  # noqa: E402

UNIT = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from wick_b200 import ops
    return ops


def borders(weights, around):
    """Uniform numbers at and beside the sums at which one thread's tokens (a 1024th of the row) end, and the smallest and largest."""
    vocab = len(weights)
    chunk = -(-vocab // 1024)
    ends = weights.cumsum(0)[torch.arange(chunk - 1, vocab, chunk).clamp(max=vocab - 1)] / weights.sum()
    at = (ends / UNIT).round().long()[:, None] + torch.arange(-around, around + 1)
    at = torch.cat([at.flatten(), torch.tensor([0, 1, 2, (1 << 24) - 1, (1 << 24) - 2])]).clamp(0, (1 << 24) - 1)
    return (at.double() * UNIT).float()


@pytest.mark.parametrize("vocab,share,around", [(32768, 0.03, 2), (151936, 0.03, 1), (100003, 0.5, 1), (1025, 0.3, 3), (5000, 0.001, 2)])
def test_a_draw_over_all_tokens_takes_an_allowed_one(ops, vocab, share, around):
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(vocab, generator=g) * 2).float()
    allowed = torch.rand(vocab, generator=g) < share
    allowed[0] = allowed[-1] = False
    allowed[vocab // 2] = True
    x[~allowed] = -math.inf
    weights = torch.exp((x - x.max()).double() / 0.9)
    u = borders(weights, around)
    got = ops.sample_temperature(x.cuda().expand(len(u), vocab).contiguous(), 0.9, u.cuda()).cpu().long()
    assert bool(allowed[got].all()), f"{int((~allowed[got]).sum())} of {len(u)} draws took a token that is ruled out"
    # ... and the one whose share of the sum holds the uniform number, as far as sums of a thread's tokens and of 1024 threads in 32 bits tell
    off = (-(-vocab // 1024) + 32) * 2.0 ** -23
    upto = weights.cumsum(0) / weights.sum()
    assert bool((upto[got] >= u.double() - off).all()) and bool((upto[got] - weights[got] / weights.sum() <= u.double() + off).all())


def test_a_draw_over_all_tokens_of_boundless_logits(ops):
    x = torch.randn((3, 5000), generator=torch.Generator().manual_seed(3))
    x[:, 17] = math.inf
    x[1:, 4000] = math.inf
    got = ops.sample_temperature(x.cuda(), 0.7, torch.tensor([0.9, 0.2, 0.8], device="cuda"))
    assert got.tolist() == [17, 17, 4000]


@pytest.mark.parametrize("temperature,min_p,top_p", [(1.0, 0.0, 1.0), (0.8, 0.05, 0.9), (3.0, 0.0, 0.999999)])
def test_a_draw_from_sorted_candidates_takes_an_allowed_one(ops, temperature, min_p, top_p):
    g = torch.Generator().manual_seed(5)
    rows, k = 20000, 40
    x = (torch.randn((rows, k), generator=g) * 2).sort(1, descending=True).values
    n = torch.randint(1, k + 1, (rows, 1), generator=g)
    x[torch.arange(k) >= n] = -math.inf
    ids = torch.rand((rows, 1000), generator=g).argsort(1)[:, :k].to(torch.int32)
    u = torch.rand(rows, generator=g)
    u[::3], u[1::3] = 1.0 - UNIT, 1.0 - 2 * UNIT
    u[0] = 0.0
    got = ops.pick_sorted(x.cuda(), ids.cuda(), u.cuda(), temperature, min_p, top_p).cpu()
    place = (ids == got[:, None]).int().argmax(1)
    bad = int((x[torch.arange(rows), place] == -math.inf).sum())
    assert bad == 0, f"{bad} of {rows} draws took a candidate that is ruled out"
    # the plain form says the same but where the exponential's last bit decides
    cfg = SamplerConfig(temperature=temperature, top_k=k, top_p=top_p, min_p=min_p)
    same = sum(int(got[i]) == pick_from_sorted(x[i].numpy(), ids[i].numpy(), cfg, type("R", (), {"next_f32": lambda s, v=float(u[i]): v})())
               for i in range(500))
    assert same >= 490


def test_a_draw_from_boundless_candidates(ops):
    x = torch.tensor([[math.inf, 3.0, -math.inf], [math.inf, math.inf, 5.0]])
    ids = torch.tensor([[4, 5, 6], [7, 8, 9]], dtype=torch.int32)
    for u, want in ((0.0, [4, 7]), (0.9, [4, 8])):
        assert ops.pick_sorted(x.cuda(), ids.cuda(), torch.full((2,), u, device="cuda"), 1.0, 0.0, 1.0).tolist() == want


def test_rules_hold_for_drawn_tokens():
    """A biased token of +inf is always drawn, tokens outside ``allowed`` never, however few are left for the candidates."""
    import wick_b200 as wick
    from helpers import make_engine
    eng = make_engine("A", "float32", max_tokens=4096)
    allowed = [3, 77, 300]
    for top_k in (0, 40):
        sampler = wick.SamplerConfig(temperature=1.5, top_k=top_k, top_p=1.0, seed=11)
        got = wick.sample_many(eng, [[1, 2, 3]], 20, wick.GenOptions(max_tokens=20, sampler=sampler, rules=wick.LogitRules(allowed=allowed)))[0]
        assert {t for r in got for t in r.tokens} == set(allowed)
        got = wick.generate(eng, [[1, 2, 3]] * 2, wick.GenOptions(max_tokens=5, sampler=sampler, rules=wick.LogitRules(bias={33: math.inf})))
        assert all(r.tokens == [33] * 5 for r in got)
    assert np.isfinite(eng.step([eng.open_seq()], [[1, 2]]).cpu().numpy()).all()
