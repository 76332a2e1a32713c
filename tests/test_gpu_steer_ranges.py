"""Bias ranges that name more than there is."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_shared_prefix import ints, ops  # noqa: E402,F401


@pytest.mark.parametrize("vocab", [70, 5000])
def test_ranges_end_with_the_entries(ops, vocab):
    x = torch.randn((3, vocab), generator=torch.Generator().manual_seed(1)).cuda()
    tokens, values = ints([3, vocab - 1, vocab, -4]), torch.tensor([1.5, -2.0, 9.0, 9.0], device="cuda")
    got = ops.steer_logits(x.clone(), bias=(ints([-7, 1, 100000, 2]), tokens, values))
    want = x.clone()
    want[0, 3] += 1.5                                            # from the first entry on
    want[1, vocab - 1] += -2.0                                   # to the last one; tokens outside the vocabulary are none
    assert torch.equal(got, want)                                # (the third range ends before it begins)
    got = ops.steer_logits(x.clone(), bias=(ints([0, 5, 5, 5]), ints([]), torch.zeros(0, device="cuda")))
    assert torch.equal(got, x)
