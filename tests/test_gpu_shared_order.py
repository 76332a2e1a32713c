"""Groups of a step that are not one behind the other: reported, whatever they would have needed of scratch."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_shared_prefix import BF16, F32, Case, ints, kernels_of, ops  # noqa: E402,F401


@pytest.mark.parametrize("pages,heads,kv_heads,dim,dtype,kernels", [(3, 8, 2, 128, BF16, 2), (3, 8, 2, 48, BF16, 2), (3, 4, 4, 64, F32, 2),
                                                                    (130, 32, 8, 128, BF16, 3), (260, 16, 4, 64, BF16, 3)])
def test_groups_in_no_order_are_reported(ops, pages, heads, kv_heads, dim, dtype, kernels):
    n, G = 12, 40
    case = Case([(pages, [(i % 5, 1) for i in range(n)])] + [(pages, [])] * (G - 1), heads, kv_heads, dim, dtype, seed=1)
    shared = ops.SharedPrefix.of(case.sizes, case.shared, case.kv_lens, "cuda")
    q, kv, b = case.q.cuda(), case.kv.cuda(), case.batch()
    # every second group has all sequences
    wrong = shared._replace(cu_groups=ints([0 if g % 2 == 0 else n for g in range(G + 1)]))
    words = ops.attention_shared_scratch(shared, b, heads, kv_heads, dim, dtype)
    scratch = torch.full((words + 4096,), 7.0, device="cuda")
    assert kernels_of(ops, lambda: ops.attention_shared(q, kv, b, wrong, case.scale, scratch[:words])) == kernels
    with pytest.raises(ops.KernelError, match="in no order"):
        ops.check_status()
    assert bool((scratch[words:] == 7.0).all()), "nothing is written beyond the scratch"
    # the next call is as ever
    got = ops.attention_shared(q, kv, b, shared, case.scale, scratch[:words])
    want, most = case.want()
    assert ((got.double().cpu() - want).abs() / most).max().item() <= 1.0
    ops.check_status()


def test_groups_beyond_the_sequences_are_cut_off(ops):
    case = Case([(3, [(10, 1), (70, 1)]), (2, [(5, 1)])], 8, 2, 128, BF16, seed=2)
    shared = ops.SharedPrefix.of(case.sizes, case.shared, case.kv_lens, "cuda")._replace(cu_groups=ints([0, 2, 900]))
    got = ops.attention_shared(case.q.cuda(), case.kv.cuda(), case.batch(), shared, case.scale)
    want, most = case.want()
    assert ((got.double().cpu() - want).abs() / most).max().item() <= 1.0
    ops.check_status()
