"""Kinds of storage that can be forked, and those that cannot say how."""
import pytest
import torch

from wick_b200.cache import Cache, Storage, register_storage
from wick_b200.parts.base import CacheNeed


class Silent(Storage):
    kind = "silent_records"

    def shape(self):
        return (self.n_entries, self.n_slots, 3)


def test_a_kind_that_says_nothing_is_not_copied_in_silence():
    register_storage("silent_records", Silent)
    try:
        c = Cache([CacheNeed("paged_kv", kv_heads=1, head_dim=4), CacheNeed("silent_records")], max_tokens=128, dtype=torch.float32, device="cpu")
    finally:
        from wick_b200.cache import cache
        del cache._STORAGE["silent_records"]
    at = torch.tensor([1])
    assert c.cannot_copy() == ["silent_records"]
    for copy in (c.copy_pages, c.copy_slots):
        with pytest.raises(NotImplementedError, match="silent_records"):
            copy(at, at + 1)


def test_the_kinds_of_the_package_can_all_be_forked():
    needs = [CacheNeed("paged_kv", kv_heads=1, head_dim=4), CacheNeed("paged_rows", shape=(3,)),
             CacheNeed("paged_blocks", kv_heads=1, head_dim=4, block=16), CacheNeed("state", shape=(2,))]
    c = Cache(needs, max_tokens=128, dtype=torch.float32, device="cpu", max_seqs=2)
    assert c.cannot_copy() == []
    c.copy_pages(torch.tensor([1]), torch.tensor([2]))
    c.copy_slots(torch.tensor([1]), torch.tensor([2]))
