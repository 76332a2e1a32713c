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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_records_have_a_bound(d, dtype):
    """New tokens of many rows behind a long cache: what lies between the two kernels stays within 256 MB, whatever the length."""
    from wick_b200 import ops
    kinds = (None, "plain") if dtype == torch.float32 else (None, "plain", "records", "stay")
    for heads, kv, new, seqs, length in ((16, 1, 2000, 1, 62000), (16, 1, 290, 1, 65000), (16, 1, 130, 1, 131000), (64, 8, 10, 16, 131000), (32, 2, 100, 3, 1000000),
                                         (24, 2, 30000, 1, 100000), (9, 1, 1, 4000, 40000), (128, 1, 1, 900, 131000)):
        b = batch(new * seqs, seqs, -(-(length + new) // 64), new, starts=[length] * seqs, q_lens=[new] * seqs)
        for kind in kinds:
            if kind == "stay" and seqs > 1024:
                continue
            if kind is None and new > 1 and new * heads // kv > ops.kv4.OPEN_ROWS.get(d, 1 << 30) and dtype == torch.bfloat16:
                continue                                             # (opened)
            assert 4 * ops.attention_kv4_scratch(b, heads, kv, d, dtype, kind=kind) <= 256 << 20, (heads, kv, new, kind)


def test_records_follow_the_length_alone_up_to_eight_rows():
    """... where a sequence's result does not depend on the batch that it is in."""
    from wick_b200 import ops
    for seqs in (1, 64, 1000):
        b = batch(seqs, seqs, 2048, 1)
        assert ops.attention_kv4_scratch(b, 8, 1, 128, torch.bfloat16, kind="records") == seqs * 8 * 128 * 130
        assert ops.attention_kv4_scratch(b, 8, 1, 128, torch.float32, kind="plain") == seqs * 8 * 1024 * 130


def test_what_a_frozen_workspace_gave():
    """A captured step keeps the scratch that it asked for, and no other's."""
    from wick_b200.engine.engine import Workspace
    w = Workspace(torch.device("cpu"))
    w.get("a", 10, torch.float32)
    b = w.get("b", 20, torch.float32)
    w.frozen, w.taken = True, {}
    assert w.get("b", 5, torch.float32) is b
    with pytest.raises(RuntimeError):
        w.get("c", 1, torch.float32)
    w.frozen = False
    w.get("a", 100, torch.float32)
    assert set(w.taken) == {"b"} and w.taken["b"] is b
