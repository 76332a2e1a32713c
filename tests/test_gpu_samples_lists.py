"""Continuations against the plain loop as whole lists of tokens."""
import pytest

pytestmark = pytest.mark.gpu

import wick_b200 as wick  # noqa: E402
from helpers import CONFIGS, make_engine, plain_model, poison_all, random_tokens  # noqa: E402
from plain import qwen3_plain as P  # noqa: E402

STD = 0.08
GREEDY = wick.SamplerConfig.greedy()


def done(eng):
    eng.cache.check()
    assert eng.cache.slots.n_held == 0 and eng.cache.pages.n_held == 0


def prompt(name, n, seed=0):
    return random_tokens(CONFIGS[name]["vocab_size"], n, 400 + seed)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_greedy_continuations_end_where_the_plain_loop_does(name, graphs):
    eng = make_engine(name, "float32", std=STD, max_tokens=8192, use_graphs=graphs)
    poison_all(eng)
    cfg, w = plain_model(name, std=STD)
    prompts = [prompt(name, n, n) for n in (5, 64, 130, 63)]
    free = [P.greedy(cfg, w, p, 9) for p in prompts]
    own = set(eng.spec.stop_token_ids)
    # a token that some prompts' continuations come to, and none
    for extra in ([], [free[0][4]], [free[1][0], free[3][8]]):
        stops = own | set(extra)
        got = wick.sample_many(eng, prompts, 2, wick.GenOptions(max_tokens=9, sampler=GREEDY, stop_token_ids=extra))
        for p, ref, rs in zip(prompts, free, got):
            cut = next((i for i, t in enumerate(ref) if t in stops), None)
            for r in rs:
                assert (r.tokens, r.finish, r.prompt_tokens) == (ref if cut is None else ref[:cut], "length" if cut is None else "stop", len(p))
    done(eng)
