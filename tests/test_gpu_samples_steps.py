"""Continuations of many prompts, and the captured steps that they are decoded by."""
import pytest

pytestmark = pytest.mark.gpu

import wick_b200 as wick  # noqa: E402
from helpers import make_engine  # noqa: E402
from test_gpu_samples_lists import GREEDY, STD, done  # noqa: E402


def test_more_prompts_than_a_step_has_groups():
    eng = make_engine("A", "float32", std=STD, max_tokens=64 * 3500)
    prompts = [[10 + i % 5, 20] for i in range(1030)]
    opts = wick.GenOptions(max_tokens=2, sampler=GREEDY, max_batch=2000)
    want = [r.tokens for r in wick.generate(eng, prompts[:5], opts)]
    got = wick.sample_many(eng, prompts, 1, opts)
    assert [rs[0].tokens for rs in got] == [want[i % 5] for i in range(1030)]
    done(eng)
