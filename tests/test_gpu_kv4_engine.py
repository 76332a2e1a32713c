"""Engines whose cache holds keys and values in 4 bits, against the plain decoder with keys and values as such a cache holds them."""
import json

import pytest
import torch

pytestmark = pytest.mark.gpu

import wick_b200 as wick  # noqa: E402
from helpers import CONFIGS, assert_logits_close, make_engine, model_dir, plain_model, random_tokens  # noqa: E402
from plain import qwen3_kv4_plain as P  # noqa: E402

STD = 0.08
GREEDY = wick.SamplerConfig.greedy()


def engine(name, dtype, **kw):
    eng = make_engine(name, dtype, std=STD, cache_bits=4, **kw)
    for g in eng.cache.groups:                                       # (numbers that are none in every place)
        assert g.need.kind == "paged_kv4"
        g.storage.fill_(255)
    return eng


def held(eng, slot, n):
    """What the cache holds of a sequence's first n positions, per layer."""
    from wick_b200 import ops
    table = torch.tensor([eng.cache.pages_of(slot)], dtype=torch.int32, device="cuda")
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    return [ops.kv4_read(kv, eng.config.head_dim, table, torch.zeros_like(at), at).double().cpu() for kv in eng.cache.groups[0].storage]


def check(eng, slot, tokens, got, rows, name, dtype, what):
    """The logits are those of the plain decoder with the keys and values that the cache holds, as near as with any cache; and the cache holds every number as
    near as a code can be (half a step of its group's range; what rounding the scales and the value adds), apart from what the
    activations' own rounding moved it by."""
    cfg, w = plain_model(name, std=STD)
    cached = held(eng, slot, len(tokens))
    want, made = P.forward(cfg, w, tokens, cached=cached)
    assert_logits_close(got, want[rows], dtype, what)
    for (k, v), c in zip(made, cached):
        for x, y in ((k, c[0]), (v, c[1])):
            x, y = x.unflatten(-1, (-1, 32)), y.unflatten(-1, (-1, 32))
            reach, top = x.amax(-1) - x.amin(-1), x.abs().amax(-1)
            bound = reach / 30 + 2.0 ** -8 * (top + 3 * reach) + (1e-4 if dtype == "float32" else 0.05) * top
            assert ((x - y).abs().amax(-1) <= bound).all(), what


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["D", "E", "F"])
def test_logits(name, dtype):
    """Whole prompts of several lengths, the same in pieces, and token by token; captured steps and others."""
    vocab = CONFIGS[name]["vocab_size"]
    for graphs in (False, True):
        eng = engine(name, dtype, use_graphs=graphs)
        for n, seed in ((1, 1), (65, 2), (200, 3)):
            toks = random_tokens(vocab, n, seed)
            s = eng.open_seq()
            check(eng, s, toks, eng.step([s], [toks], [list(range(n))]), range(n), name, dtype, (name, n, "whole"))
            eng.truncate_seq(s, n // 2)
            pos, got = n // 2, []
            for size in (1, 1, 3, 1, 17, 1, 40):
                if pos + size <= n:
                    got.append(eng.step([s], [toks[pos:pos + size]], [list(range(size))]).clone())
                    pos += size
            if got:
                check(eng, s, toks[:pos], torch.cat(got), range(n // 2, pos), name, dtype, (name, n, "pieces"))
            eng.close_seq(s)
        # unequal sequences together, their first steps and the next ones
        lens = (5, 130, 64, 1)
        toks = [random_tokens(vocab, n + 4, 50 + n) for n in lens]
        slots = [eng.open_seq() for _ in lens]
        got = [eng.step(slots, [t[:n] for t, n in zip(toks, lens)]).clone()]
        got += [eng.step(slots, [[t[n + i]] for t, n in zip(toks, lens)]).clone() for i in range(4)]
        for b, n in enumerate(lens):
            check(eng, slots[b], toks[b], torch.stack([g[b] for g in got]), range(n - 1, n + 4), name, dtype, (name, n, "batch"))
            eng.close_seq(slots[b])
        eng.check_kernels()
        eng.cache.check()


def test_bytes():
    for name, kv, d, layers in (("D", 2, 64, 2), ("E", 1, 128, 2)):
        eng, wide = engine(name, "bfloat16"), make_engine(name, "bfloat16", std=STD)
        assert eng.cache.bytes_per_token() == layers * kv * 2 * d * 5 // 8
        assert wide.cache.storage_bytes() * 5 == eng.cache.storage_bytes() * 16
        assert eng.cache.read_bytes(100, 3) == 100 * eng.cache.bytes_per_token()


@pytest.mark.parametrize("name", ["D", "E"])
def test_generate_and_samples(name):
    """Greedy tokens of the plain loop, as long as its best logit is clearly the best; continuations of a prompt over one copy of its cache are the same."""
    cfg, w = plain_model(name, std=STD)
    vocab = CONFIGS[name]["vocab_size"]
    prompts = [random_tokens(vocab, n, 70 + n) for n in (3, 64, 90)]
    want = [P.greedy(cfg, w, p, 8) for p in prompts]
    eng = engine(name, "float32", max_tokens=4096)
    opts = wick.GenOptions(max_tokens=8, sampler=GREEDY)
    once = wick.generate(eng, prompts, opts)
    for g in eng.cache.groups:
        g.storage.fill_(255)
    many = wick.sample_many(eng, prompts, 3, opts)
    for p, (tokens, lead), one, some in zip(prompts, want, once, many):
        scale = P.forward(cfg, w, p).abs().max()
        sure = next((i for i, x in enumerate(lead) if x < 0.02 * scale), 8)
        assert one.tokens[:sure] == tokens[:sure]
        assert all(r.tokens[:sure] == tokens[:sure] for r in some)
    assert eng.cache.pages.n_held == 0 and eng.cache.slots.n_held == 0
    # (in bfloat16 products of another number of rows round in another order, and a code that changes is a larger step: the same call gives the same)
    eng = engine(name, "bfloat16")
    first = [r.tokens for r in wick.generate(eng, prompts, opts)]
    assert all(len(t) == 8 for t in first) and [r.tokens for r in wick.generate(eng, prompts, opts)] == first


def test_refusals():
    with pytest.raises(ValueError, match="head sizes"):
        make_engine("B", "bfloat16", cache_bits=4)
    with pytest.raises(ValueError, match="8 bits"):
        make_engine("D", "bfloat16", cache_bits=8)
    from test_nibotar_config import CONFIG
    with pytest.raises(ValueError, match="do not keep their cache in 4 bits"):
        wick.Engine.from_config(wick.config_from_json(CONFIG), 1, cache_bits=4)


def test_command_line(capsys):
    from wick_b200 import cli
    d = model_dir("D", std=STD)
    assert cli.main(["run", d, "--ids", "5,17,3", "-n", "5", "-t", "0", "--cache-bits", "4"]) == 0
    out = capsys.readouterr()
    assert len(json.loads(out.out.splitlines()[0])) == 5 and "in 4 bits" in out.err
    assert cli.main(["run", d, "--ids", "5", "--cache-bits", "3"]) == 2
