"""The cache in 4 bits, what needs no device: scratch and what is kept between calls."""
import types

import pytest
import torch


def batch(n_tokens, n_seqs, pages, max_q, **kw):
    return types.SimpleNamespace(n_tokens=n_tokens, n_seqs=n_seqs, table_width=pages, max_q_len=max_q, kv_bound=64 * pages, **kw)


def test_plans_are_kept_for_each_device(monkeypatch):
    """The number of multiprocessors decides how a step is cut: what is kept for one device does not answer for another."""
    from wick_b200 import ops
    from wick_b200.ops import kv4
    here, asked = [0], []

    def scratch(*sizes):
        asked.append(here[0])
        return 1000 * (here[0] + 1)
    monkeypatch.setattr(kv4, "_device", lambda: here[0])
    monkeypatch.setattr(kv4, "_kv4", lambda d: types.SimpleNamespace(_lib=types.SimpleNamespace(wick_attn_kv4_scratch=scratch)))
    kv4._plan.cache_clear()
    try:
        b = batch(3, 2, 700, 2)
        for device in (0, 1, 0, 1):
            here[0] = device
            assert ops.attention_kv4_scratch(b, 8, 2, 128, torch.bfloat16, kind="records") == 1000 * (device + 1)
        assert asked == [0, 1]
    finally:
        kv4._plan.cache_clear()
