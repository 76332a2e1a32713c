"""Continuations of models whose caches keep other things than keys and values."""
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

import test_gpu_fasunex as fasunex  # noqa: E402
import test_gpu_kikopel as kikopel  # noqa: E402
import test_gpu_nibotar as nibotar  # noqa: E402
import test_gpu_saposun as saposun  # noqa: E402
import test_gpu_sunosun as sunosun  # noqa: E402
import test_gpu_toy_parts as toy  # noqa: E402
import test_gpu_tuguvik as tuguvik  # noqa: E402
import wick_b200 as wick  # noqa: E402
from helpers import CONFIG_B, random_tokens, tmp_root  # noqa: E402
from test_gpu_samples_lists import GREEDY, done  # noqa: E402
from wick_b200.cache import register_storage  # noqa: E402


def toy_engine(graphs):
    cfg = wick.config_from_json(dict(CONFIG_B, architectures=["ToyWindowForCausalLM"]))
    d = os.path.join(tmp_root(), "toy-window-samples")
    wick.write_random_model(cfg, 8, d, dtype=torch.float32)
    return wick.Engine.from_dir(d, dtype="float32", max_tokens=2048, use_graphs=graphs)


def test_a_storage_that_says_nothing_of_copies_is_refused():
    eng = toy_engine(True)
    with pytest.raises(RuntimeError, match="toy_last_rows"):
        wick.sample_many(eng, [[1, 2, 3]], 2, wick.GenOptions(max_tokens=3, sampler=GREEDY))
    done(eng)
    # what the model could do before it still does
    assert len(wick.generate(eng, [[1, 2, 3]], wick.GenOptions(max_tokens=3, sampler=GREEDY))[0].tokens) <= 3


class CopiedRows(toy.LastRows):
    def copy_pages(self, src, dst):
        pass

    def copy_slots(self, src, dst):
        self.tensor[:, dst] = self.tensor[:, src]


@pytest.mark.parametrize("graphs", [True, False])
def test_a_storage_of_ones_own_that_copies_its_records(graphs):
    register_storage("toy_last_rows", CopiedRows)
    try:
        eng = toy_engine(graphs)
    finally:
        register_storage("toy_last_rows", toy.LastRows)
    prompts = [random_tokens(1000, n, n) for n in (70, 3, 64)]
    opts = lambda seed: wick.GenOptions(max_tokens=9, sampler=wick.SamplerConfig(temperature=0.8, top_k=30, seed=seed))   # noqa: E731
    got = wick.sample_many(eng, prompts, 3, opts(7))
    for i, p in enumerate(prompts):
        for k in range(3):
            assert got[i][k].tokens == wick.generate(eng, [p], opts(7 + k))[0].tokens
    done(eng)


FAMILIES = [(m, name) for m in (fasunex, kikopel, nibotar, saposun, sunosun, tuguvik) for name in sorted(m.CONFIGS)]


@pytest.mark.parametrize("family,name", FAMILIES, ids=[n for _, n in FAMILIES])
def test_continuations_of_every_family_are_what_each_draws_alone(family, name):
    """Keys and values, latent rows, pooled blocks and records of a sequence: whatever a family keeps is shared or copied."""
    eng = family.engine(name, "float32", max_tokens=8192)
    prompts = [random_tokens(eng.spec.vocab, n, n) for n in (70, 12, 130)]
    opts = lambda seed: wick.GenOptions(max_tokens=8, sampler=wick.SamplerConfig(temperature=0.7, top_k=10, seed=seed))   # noqa: E731
    got = wick.sample_many(eng, prompts, 3, opts(7))
    for i, p in enumerate(prompts):
        for k in range(3):
            assert got[i][k].tokens == wick.generate(eng, [p], opts(7 + k))[0].tokens
    done(eng)
