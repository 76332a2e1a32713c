"""Continuations of many prompts, and the captured steps that they are decoded by."""
import pytest

pytestmark = pytest.mark.gpu

import wick_b200 as wick  # noqa: E402
from helpers import make_engine, plain_model  # noqa: E402
from plain import qwen3_plain as P  # noqa: E402
from test_gpu_samples_lists import GREEDY, STD, done, prompt  # noqa: E402


def test_more_prompts_than_a_step_has_groups():
    eng = make_engine("A", "float32", std=STD, max_tokens=64 * 3500)
    prompts = [[10 + i % 5, 20] for i in range(1030)]
    opts = wick.GenOptions(max_tokens=2, sampler=GREEDY, max_batch=2000)
    want = [r.tokens for r in wick.generate(eng, prompts[:5], opts)]
    got = wick.sample_many(eng, prompts, 1, opts)
    assert [rs[0].tokens for rs in got] == [want[i % 5] for i in range(1030)]
    done(eng)


def test_captured_steps_are_bounded_and_a_batch_that_shrinks_keeps_its_own(monkeypatch):
    from wick_b200.engine import engine as E
    eng = make_engine("B", "float32", std=STD, max_tokens=64 * 400)
    cfg, w = plain_model("B", std=STD)
    p = prompt("B", 66)
    opts = lambda stops=(): wick.GenOptions(max_tokens=30, sampler=wick.SamplerConfig(temperature=1.0, top_k=50, seed=3), stop_token_ids=stops)   # noqa: E731
    free = wick.sample_many(eng, [p], 6, opts())[0]
    assert len(eng._shared_graphs) == 1
    # continuations that end one after the other, at different lengths
    stops = [free[2].tokens[4], free[0].tokens[9], free[5].tokens[12]]
    got = wick.sample_many(eng, [p], 6, opts(stops))[0]
    for f, r in zip(free, got):
        cut = next((i for i, t in enumerate(f.tokens) if t in stops), None)
        assert r.tokens == (f.tokens if cut is None else f.tokens[:cut])
    assert len(eng._shared_graphs) == 1, "a short rest of a batch is decoded by the step that is there"
    # another number of prompts is no other step while a power of two holds it
    many = [prompt("B", 66, s) for s in range(7)]
    want = [P.greedy(cfg, w, q, 5) for q in many]
    own = set(eng.spec.stop_token_ids)
    cut = [t[:next((i for i, x in enumerate(t) if x in own), 5)] for t in want]
    greedy = wick.GenOptions(max_tokens=5, sampler=GREEDY)
    for n in (4, 5, 6, 7):
        assert [[r.tokens for r in rs] for rs in wick.sample_many(eng, many[:n], 1, greedy)] == [[t] for t in cut[:n]]
    assert len(eng._shared_graphs) <= 4 and all(k[2] & (k[2] - 1) == 0 for k in eng._shared_graphs)
    # the oldest make room
    monkeypatch.setattr(E, "SHARED_GRAPH_COUNT", 2)
    for n in (1, 2, 5, 1, 9, 20, 2):
        assert [r.tokens for r in wick.sample_many(eng, [many[0]], n, greedy)[0]] == [cut[0]] * n
        assert len(eng._shared_graphs) <= 4
    for n in (1, 2, 5, 9, 20):
        wick.sample_many(eng, [many[0]], n, greedy)
        wick.sample_many(eng, [many[0]], n, wick.GenOptions(max_tokens=80, sampler=GREEDY))
    assert len(eng._shared_graphs) <= 2
    done(eng)
