"""Rules on the logits and pages lent to a batch: what needs no GPU."""
import pytest
import torch

import wick_b200 as wick
from wick_b200 import cli
from wick_b200.cache import Cache, CacheFull, PoolError
from wick_b200.engine.samples import pages_of_batch
from wick_b200.parts.base import CacheNeed


def test_rules_are_checked():
    wick.LogitRules(0.5, -0.5, {0: 1.0, 9: -float("inf")}, [0, 9]).check(10)
    for bad, text in ((wick.LogitRules(bias={10: 1.0}), "token id 10 of bias"), (wick.LogitRules(allowed=[-1]), "token id -1 of allowed"),
                      (wick.LogitRules(bias={1: float("nan")}), "not a number"), (wick.LogitRules(allowed=[]), "no token"),
                      (wick.LogitRules(frequency_penalty=float("inf")), "frequency_penalty"), (wick.LogitRules(presence_penalty=float("nan")), "presence_penalty")):
        with pytest.raises(ValueError, match=text):
            bad.check(10)


def test_rules_need_a_device_run():
    class Engine:
        cache = Cache([], max_tokens=640, dtype=torch.float32, device="cpu", allocate=False)

        def open_seq(self):
            return self.cache.open_seq()

    with pytest.raises(ValueError, match="on the device"):
        wick.generate(Engine(), [[1]], wick.GenOptions(max_tokens=2, rules=wick.LogitRules()))


def test_lent_pages_are_held_by_nobody_until_they_come_back():
    c = Cache([CacheNeed("paged_kv", kv_heads=1, head_dim=16)], max_tokens=640, dtype=torch.float32, device="cpu", allocate=False)
    s = c.open_seq()
    c.reserve(s, 100)
    pages = c.lend(5)
    c.check()
    assert len(set(pages)) == 5 and 0 not in pages and not set(pages) & set(c.pages_of(s)) and c.pages.n_free == 3
    with pytest.raises(CacheFull, match="4 pages"):
        c.lend(4)
    c.give_back(pages[:2])
    c.check()
    with pytest.raises(PoolError, match="not lent"):
        c.give_back(pages[:1])
    with pytest.raises(PoolError, match="not lent"):
        c.give_back(c.pages_of(s)[:1])
    c.give_back(pages[2:])
    c.close_seq(s)
    c.check()
    assert c.pages.n_held == 0


def test_copies_of_pages_and_records():
    needs = [CacheNeed("paged_kv", kv_heads=2, head_dim=4), CacheNeed("paged_rows", shape=(3,)), CacheNeed("state", shape=(2, 5))]
    c = Cache(needs * 2, max_tokens=256, dtype=torch.float32, device="cpu", max_seqs=4)
    for g in c.groups:
        g.storage.normal_()
    before = [g.storage.clone() for g in c.groups]
    at = lambda *v: torch.tensor(v)      # noqa: E731
    c.copy_pages(at(1, 1, 4), at(2, 3, 1))
    c.copy_slots(at(1, 1), at(3, 4))
    for g, b in zip(c.groups, before):
        want = b.clone()
        if g.need.kind == "state":
            want[:, 3], want[:, 4] = b[:, 1], b[:, 1]
        else:
            want[:, 2], want[:, 3], want[:, 1] = b[:, 1], b[:, 1], b[:, 4]
        assert torch.equal(g.storage, want)


def test_pages_of_a_batch():
    assert pages_of_batch(64, 10, 3) == 1 + 3 * 2            # nothing behind the whole pages: 10 tokens on a page, and one more
    assert pages_of_batch(65, 64, 1) == 2 + 3                # one position of the prompt and 64 tokens: two pages
    assert pages_of_batch(3, 1, 2) == 1 + 2 * 2


def test_command_line_options_for_rules_and_samples():
    a = cli.parse_args(["run", "d", "--samples", "4", "--frequency-penalty", "0.5", "--presence-penalty", "-0.25", "--logit-bias", "3:1.5,4:-2", "--allow", "1,2",
                        "--allow", "7"])
    assert a.samples == 4 and a.rules == {"frequency_penalty": 0.5, "presence_penalty": -0.25, "bias": {3: 1.5, 4: -2.0}, "allowed": [1, 2, 7]}
    for bad in (["--samples", "0"], ["--logit-bias", "3"], ["--logit-bias", "a:1"], ["--allow", "x"], ["--frequency-penalty", "x"]):
        with pytest.raises(cli.UsageError):
            cli.parse_args(["run", "d"] + bad)
