"""Attention over a shared prefix: many new tokens a sequence, wide groups of heads with long own keys, head sizes beyond the usual ones."""
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_shared_prefix import BF16, F32, Case, check, kernels_of, ops  # noqa: E402,F401


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (48, BF16), (64, F32)])
def test_hundreds_of_new_tokens(ops, dim, dtype):
    case = Case([(2, [(0, 200), (77, 1), (64, 333)]), (0, [(3, 130)]), (5, [(10, 65), (1, 0)])], 8, 2, dim, dtype, seed=dim, more_width=2)
    check(case.run(ops), case)
    ops.check_status()


@pytest.mark.parametrize("dim", [64, 128])
def test_hundreds_of_new_tokens_behind_a_long_prefix(ops, dim):
    case = Case([(90 * 128 // dim, [(0, 150), (70, 260), (5, 1)])], 16, 4, dim, BF16, seed=dim)
    assert kernels_of(ops, lambda: check(case.run(ops), case)) == 3
    ops.check_status()


@pytest.mark.parametrize("heads,kv_heads", [(32, 2), (48, 3), (33, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_wide_groups_of_heads_with_long_own_keys(ops, dim, heads, kv_heads):
    case = Case([(200 * 128 // dim, [(900, 1), (3, 1), (2100, 1), (640, 1)] * 3), (0, [(300, 1)])], heads, kv_heads, dim, BF16, seed=heads + dim)
    assert kernels_of(ops, lambda: check(case.run(ops), case)) == 3
    ops.check_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [80, 96, 112, 176, 256])
def test_other_head_sizes(ops, dim, dtype):
    case = Case([(4, [(17, 1), (300, 1), (64, 5)]), (0, [(70, 1)]), (11, [(1, 1)] * 9)], 6, 2, dim, dtype, seed=dim, more_width=1)
    check(case.run(ops), case)
    ops.check_status()
