"""Attention over a shared prefix: the rounding of the weights that count cancels against their sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_shared_prefix import BF16, Case, kernels_of, ops  # noqa: E402,F401


@pytest.mark.parametrize("dim", [48, 64, 128])
@pytest.mark.parametrize("rise", [0.0, 4.0, 30.0])
@pytest.mark.parametrize("pages,n", [(5, 6), (9, 40)])
def test_rows_of_equal_values_keep_them(ops, pages, n, rise, dim):
    """Where all values of a column are one number, the result is that number: weights rounded to bfloat16 cancel against their own sum
    (rise: how far the scores rise along the prefix, in units of log2 e).  The sums' own errors are at most (keys + 8) 2^-23 of the number,
    2^-12 here, and half of the result's last place is no less than 2^-9 of it: nothing is rounded to another number."""
    case = Case([(pages, [(i * 7 % 40, 1) for i in range(n)])], 32, 8, dim, BF16, seed=pages + n, sharp=1.0)
    u = torch.zeros(dim)
    u[::2] = 1.0
    case.q = (case.q.float() * 0.3 + u).to(BF16)
    for j, page in enumerate(case.tables[0][:pages]):
        # (score: scale * dim / 2 per unit of u in both)
        case.kv[page, 0] = (case.kv[page, 0].float() * 0.5 + u * (rise * 0.6931 * j / pages * 2 / (dim * case.scale))).to(BF16)
    column = (1.0 + torch.arange(dim) / dim).to(BF16)
    case.kv[:, 1] = torch.where(torch.isnan(case.kv[:, 1]), case.kv[:, 1], column)
    got = {}
    assert kernels_of(ops, lambda: got.update(y=case.run(ops))) == 2
    assert torch.equal(got["y"].cpu(), column.expand(n, 32, dim))
    ops.check_status()


@pytest.mark.parametrize("dim", [48, 64, 128])
@pytest.mark.parametrize("pages,n", [(5, 6), (130, 5), (130, 40)])
def test_one_key_above_the_maximum_that_the_sums_are_scaled_by(pages, n, dim, ops):
    """Two keys hold all the weight: one of the first block, and one of a block soon after it whose score is higher, by less than what makes the
    running maximum of long prefixes follow.  The weight of the second is 2^(0.5 .. 7), rounded to bfloat16, and nothing averages its rounding
    out: it cancels where a block's largest weight is summed as it is multiplied.  The others are below 2^-50 together; sums as above."""
    pages = pages * (128 // dim if pages > 9 else 1)
    case = Case([(pages, [(i * 7 % 40, 1) for i in range(n)])], 32, 8, dim, BF16, seed=pages + n)
    u = torch.zeros(dim)
    u[::2] = 1.0
    rows = torch.linspace(0.25, 3.5, n * 32).to(BF16).float()
    case.q = (rows[:, None] * u).view(n, 32, dim).to(BF16)
    unit = 2 / (dim * case.scale) / 1.4427                      # of a key along u: a score of one unit of log2 e for a query of 1
    keys = torch.where(torch.isnan(case.kv[:, 0]), case.kv[:, 0], (-200.0 * unit * u).to(BF16))
    keys[case.tables[0][0], :, 5] = 0.0
    keys[case.tables[0][2], :, 60] = (2.0 * unit * u).to(BF16)
    case.kv[:, 0] = keys
    column = (1.0 + torch.arange(dim) / dim).to(BF16)
    case.kv[:, 1] = torch.where(torch.isnan(case.kv[:, 1]), case.kv[:, 1], column)
    got = case.run(ops).cpu()
    wrong = (got != column).float().mean().item()
    assert wrong == 0.0, f"{100 * wrong:.1f} % of the results are not the values' own number"
    ops.check_status()
