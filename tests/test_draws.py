"""The plain form of the cuts and the draw where candidates are ruled out (-inf) or boundless (+inf)."""
import numpy as np
import pytest

from wick_b200.sampling.sampler import SamplerConfig, pick_from_sorted


class Fixed:
    def __init__(self, u):
        self.u = u

    def next_f32(self):
        return self.u


LAST = 1.0 - 2.0 ** -24


def candidates(rng, k, ruled_out):
    v = np.sort(rng.normal(0, 2, k).astype(np.float32))[::-1].copy()
    v[k - ruled_out:] = -np.inf
    return v, rng.permutation(10 * k)[:k].astype(np.int32)


@pytest.mark.parametrize("cfg", [SamplerConfig(temperature=1.0, top_k=0, top_p=1.0), SamplerConfig(temperature=0.8, top_p=0.9, min_p=0.05),
                                 SamplerConfig(temperature=2.5, top_p=1.0, min_p=0.001)])
def test_a_ruled_out_candidate_is_never_drawn(cfg):
    rng = np.random.default_rng(1)
    for i in range(3000):
        k = int(rng.integers(2, 41))
        v, ids = candidates(rng, k, int(rng.integers(1, k)))
        pick = pick_from_sorted(v, ids, cfg, Fixed([0.0, LAST, LAST - 2.0 ** -24, float(rng.random())][i % 4]))
        assert v[list(ids).index(pick)] > -np.inf


def test_boundless_candidates_share_the_draw():
    v, ids = np.array([np.inf, np.inf, 3.0, -np.inf], dtype=np.float32), np.array([7, 2, 9, 1], dtype=np.int32)
    cfg = SamplerConfig(temperature=1.0, top_p=1.0)
    assert [pick_from_sorted(v, ids, cfg, Fixed(u)) for u in (0.0, 0.3, 0.7, LAST)] == [7, 7, 2, 2]


def test_without_rules_the_last_candidate_ends_the_walk_as_before():
    """Finite candidates: what the walk leaves over goes to the last of those kept, even where its weight has become zero."""
    v, ids = np.array([0.0, -0.1, -500.0], dtype=np.float32), np.array([4, 5, 6], dtype=np.int32)
    f = np.float32
    p = np.exp(v - v[0]).astype(f)
    total = f(0)
    for x in p:
        total = f(total + x)
    p = (p / total).astype(f)
    tot = f(0)
    for x in p:
        tot = f(tot + x)
    r = f(f(LAST) * tot)
    for x in p:
        r = f(r - x)
    want = 6 if r > 0 else 5
    assert pick_from_sorted(v, ids, SamplerConfig(temperature=1.0, top_p=1.0), Fixed(LAST)) == want
