"""Batches of continuations that take turns on one engine."""
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_samples_lists import GREEDY, STD, done, prompt  # noqa: E402
from helpers import make_engine, plain_model  # noqa: E402
from plain import qwen3_plain as P  # noqa: E402
from wick_b200.engine.samples import SampleRun  # noqa: E402


@pytest.mark.parametrize("graphs", [True, False])
def test_two_batches_on_one_engine_taken_in_turn(graphs):
    """Both decode by the same captured step: each finds its own description there, whoever ran before."""
    eng = make_engine("A", "float32", std=STD, max_tokens=4096, use_graphs=graphs)
    cfg, w = plain_model("A", std=STD)
    prompts = [prompt("A", 70, s) for s in (1, 2)]
    runs = [SampleRun(eng, GREEDY) for _ in prompts]
    out = [[], []]
    for run, p in zip(runs, prompts):
        run.start([p], [[0, 1, 2]], [9])
    for i, run in enumerate(runs):
        out[i].append(run.collect())
    for _ in range(8):
        for i, run in enumerate(runs):
            run.launch([0, 1, 2])
            out[i].append(run.collect())
    for run in runs:
        run.close()
    for p, steps in zip(prompts, out):
        assert steps == [[t] * 3 for t in P.greedy(cfg, w, p, 9)]
    done(eng)
