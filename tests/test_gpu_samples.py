"""Several continuations of a prompt over one copy of its cache, and rules on the logits, against the plain implementation."""
import json
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import test_gpu_sunosun as sunosun  # noqa: E402
import wick_b200 as wick  # noqa: E402
from helpers import BF16_REL, CONFIGS, make_engine, model_dir, plain_model, poison_all, random_tokens  # noqa: E402
from plain import qwen3_plain as P  # noqa: E402

STD = 0.08          # (separates the top logits: the greedy token does not hang on the order of sums)
GREEDY = wick.SamplerConfig.greedy()


def prompts_for(name, lengths, seed=0):
    return [random_tokens(CONFIGS[name]["vocab_size"], n, 900 + seed + n) for n in lengths]


def plain_rules(cfg, w, prompt, n, rules, repetition=1.0, stop=()):
    """Greedy decoding by the plain model under rules, in 64 bits from its logits on."""
    seq, out = list(prompt), []
    for _ in range(n):
        x = P.forward(cfg, w, seq)[-1].double()
        for t in set(seq):
            x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
        for t in set(out):
            x[t] -= rules.frequency_penalty * out.count(t) + rules.presence_penalty
        for t, b in rules.bias.items():
            x[t] += b
        if rules.allowed is not None:
            keep = torch.zeros(len(x), dtype=torch.bool)
            keep[list(rules.allowed)] = True
            x[~keep] = -math.inf
        t = int(x.argmax())
        if t in stop:
            break
        out.append(t)
        seq.append(t)
    return out


def done(eng):
    eng.cache.check()
    assert eng.cache.slots.n_held == 0 and eng.cache.pages.n_held == 0


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_greedy_continuations_are_the_plain_loops(name):
    eng = make_engine(name, "float32", std=STD, max_tokens=4096)
    poison_all(eng)
    cfg, w = plain_model(name, std=STD)
    prompts = prompts_for(name, (5, 64, 130, 63, 128))
    want = [P.greedy(cfg, w, p, 9) for p in prompts]
    got = wick.sample_many(eng, prompts, 3, wick.GenOptions(max_tokens=9, sampler=GREEDY))
    for p, r, g in zip(prompts, want, got):
        for one in g:
            assert one.tokens == [t for t in r][:len(one.tokens)] and one.prompt_tokens == len(p)
            assert one.finish == ("length" if len(one.tokens) == 9 else "stop")
    done(eng)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name,lengths", [("D", (200, 30, 64)), ("E", (300, 1000)), ("F", (129, 5))])
def test_bfloat16_continuations_pick_what_the_plain_model_rates_best(name, lengths, graphs):
    eng = make_engine(name, "bfloat16", std=STD, max_tokens=8192, use_graphs=graphs)
    poison_all(eng)
    cfg, w = plain_model(name, std=STD)
    prompts = prompts_for(name, lengths)
    n = 70 if name == "D" else 6                          # (70: own keys pass a page's end)
    got = wick.sample_many(eng, prompts, 5, wick.GenOptions(max_tokens=n, sampler=GREEDY))
    for p, rs in zip(prompts, got):
        for r in rs[::4]:
            assert len(r.tokens) == n
            ref = P.forward(cfg, w, list(p) + r.tokens)
            for i, t in enumerate(r.tokens):
                row = ref[len(p) - 1 + i]
                assert float(row[t]) >= float(row.max()) - BF16_REL * float(row.abs().max())
    done(eng)


def test_continuation_k_draws_as_a_sequence_of_seed_plus_k_does():
    eng = make_engine("B", "float32", std=STD, max_tokens=4096)
    prompts = prompts_for("B", (70, 9))
    opts = lambda seed: wick.GenOptions(max_tokens=12, sampler=wick.SamplerConfig(temperature=0.8, top_k=20, seed=seed))   # noqa: E731
    got = wick.sample_many(eng, prompts, 4, opts(100))
    for i, p in enumerate(prompts):
        for k in range(4):
            alone = wick.generate(eng, [p], opts(100 + k))[0]
            assert got[i][k].tokens == alone.tokens and got[i][k].finish == alone.finish
    assert len({tuple(r.tokens) for r in got[0]}) > 1, "the continuations differ"
    # whatever is decoded beside it, and in however many batches
    for more in (dict(max_batch=3), dict(max_batch=1)):
        o = opts(100)
        o.max_batch = more["max_batch"]
        again = wick.sample_many(eng, prompts, 4, o)
        assert [[r.tokens for r in rs] for rs in again] == [[r.tokens for r in rs] for rs in got]
    done(eng)


RULES = {
    "penalties": wick.LogitRules(frequency_penalty=0.7, presence_penalty=0.4),
    "bias": wick.LogitRules(bias={3: 2.0, 17: -1.5, 100: 1.0}),
    "allowed": wick.LogitRules(allowed=list(range(5, 200, 3))),
    "all": wick.LogitRules(frequency_penalty=0.3, presence_penalty=-0.2, bias={8: 1.5, 50: -3.0}, allowed=list(range(0, 500, 2))),
}


@pytest.mark.parametrize("repetition", [1.0, 1.3])
@pytest.mark.parametrize("which", sorted(RULES))
def test_rules_of_generate_and_of_sample_many(which, repetition):
    eng = make_engine("A", "float32", std=STD, max_tokens=4096)
    cfg, w = plain_model("A", std=STD)
    rules = RULES[which]
    sampler = wick.SamplerConfig(temperature=0.0, repetition_penalty=repetition)
    prompts = prompts_for("A", (5, 70))
    want = [plain_rules(cfg, w, p, 10, rules, repetition) for p in prompts]
    opts = wick.GenOptions(max_tokens=10, sampler=sampler, rules=rules)
    assert [r.tokens for r in wick.generate(eng, prompts, opts)] == want
    assert [[r.tokens for r in rs] for rs in wick.sample_many(eng, prompts, 2, opts)] == [[t, t] for t in want]
    # a prompt's own rules, and none for the other one
    none = plain_rules(cfg, w, prompts[1], 10, wick.LogitRules(), repetition)
    got = wick.sample_many(eng, prompts, 2, wick.GenOptions(max_tokens=10, sampler=sampler), rules=[rules, None])
    assert [[r.tokens for r in rs] for rs in got] == [[want[0]] * 2, [none] * 2]
    done(eng)


def test_continuations_that_stop_leave_and_the_others_go_on():
    eng = make_engine("B", "float32", std=STD, max_tokens=4096)
    p = prompts_for("B", (66,))[0]
    opts = lambda stops=(): wick.GenOptions(max_tokens=30, sampler=wick.SamplerConfig(temperature=1.0, top_k=50, seed=3), stop_token_ids=stops)   # noqa: E731
    free = wick.sample_many(eng, [p], 6, opts())[0]
    stop = free[2].tokens[4]
    got = wick.sample_many(eng, [p], 6, opts([stop]))[0]
    for f, g in zip(free, got):
        cut = f.tokens.index(stop) if stop in f.tokens else len(f.tokens)
        assert g.tokens == f.tokens[:cut] and g.finish == ("stop" if stop in f.tokens else f.finish)
    assert got[2].finish == "stop" and len(got[2].tokens) <= 4
    done(eng)


@pytest.mark.parametrize("name", ["SA", "SB"])
def test_a_model_with_per_sequence_state_is_forked_with_it(name):
    """Layers that keep a record per sequence, attention by other kernels: each continuation starts from a copy."""
    eng = sunosun.engine(name, "float32", max_tokens=4096)
    prompts = [random_tokens(eng.spec.vocab, n, n) for n in (70, 12)]
    opts = lambda seed: wick.GenOptions(max_tokens=8, sampler=wick.SamplerConfig(temperature=0.7, top_k=10, seed=seed))   # noqa: E731
    got = wick.sample_many(eng, prompts, 3, opts(7))
    for i, p in enumerate(prompts):
        for k in range(3):
            assert got[i][k].tokens == wick.generate(eng, [p], opts(7 + k))[0].tokens
    done(eng)


def test_sample_many_refuses_and_leaves_the_cache_as_it_was():
    eng = make_engine("A", "float32", std=STD, max_tokens=64 * 6)
    with pytest.raises(ValueError, match="at least 1"):
        wick.sample_many(eng, [[1, 2]], 0)
    with pytest.raises(ValueError, match="empty prompt"):
        wick.sample_many(eng, [[1], []], 2)
    with pytest.raises(ValueError, match="one set of rules"):
        wick.sample_many(eng, [[1], [2]], 2, rules=[None])
    with pytest.raises(RuntimeError, match="cache pages"):
        wick.sample_many(eng, [[1] * 100], 5, wick.GenOptions(max_tokens=20))
    with pytest.raises(ValueError, match="outside the vocabulary"):
        wick.sample_many(eng, [[1, 2]], 2, wick.GenOptions(max_tokens=4, rules=wick.LogitRules(bias={512: 1.0})))
    with pytest.raises(ValueError, match="no token is allowed"):
        wick.generate(eng, [[1, 2]], wick.GenOptions(max_tokens=4, rules=wick.LogitRules(allowed=[])))
    for s in list(eng.cache.seqs):
        eng.close_seq(s)
    done(eng)
    got = wick.sample_many(eng, [[1, 2, 3]], 2, wick.GenOptions(max_tokens=0))
    assert [[r.tokens for r in rs] for rs in got] == [[[], []]]
    done(eng)


def test_command_line_samples_under_rules(capsys):
    from wick_b200 import cli
    d = model_dir("A", std=STD)
    cfg, w = plain_model("A", std=STD)
    assert cli.main(["run", d, "--ids", "5,17,3", "-n", "6", "-t", "0", "-q", "f32", "--samples", "3", "--allow", "4,8,15,16,23,42",
                     "--logit-bias", "8:0.5,42:-0.25", "--frequency-penalty", "0.25", "--presence-penalty", "0.1"]) == 0
    lines = [json.loads(x) for x in capsys.readouterr().out.strip().splitlines()]
    want = plain_rules(cfg, w, [5, 17, 3], 6, wick.LogitRules(0.25, 0.1, {8: 0.5, 42: -0.25}, [4, 8, 15, 16, 23, 42]))
    assert lines == [want] * 3
