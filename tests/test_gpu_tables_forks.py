"""Forks in step_tables: of records that are forked themselves in the same call, and those that cannot be."""
import random

import pytest

pytestmark = pytest.mark.gpu

from test_gpu_shared_prefix import PAGE, ops, pages_for, plain_tables, run_tables  # noqa: E402,F401

NAMES = ("page_table", "cu_seqlens", "kv_len", "positions", "seq_of_token", "slot_map", "head_out", "tables")


def both(ops, *a):
    for name, got, want in zip(NAMES, run_tables(ops, *a), plain_tables(*a)):
        assert got == want, name
    ops.check_status()


def test_two_sequences_change_places(ops):
    tables = [[0] * 4, [11, 12, 13, 0], [21, 22, 23, 24]]
    for _ in range(20):
        both(ops, [192, 128], [1, 70], [1, 2], tables, [31, 32, 33, 34], 0, 4, 71, [2, 1])


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("n", [3, 40, 700])
def test_forks_start_from_the_pages_that_a_record_held_before_the_call(ops, n, seed):
    """Chains, circles and parents that grow: what a parent gets or takes over in the call itself is not its children's."""
    rng = random.Random(100 * n + seed)
    width = 130
    slots = rng.sample(range(1, n + 3), n)
    held = {s: rng.randint(1, width - 8) for s in slots}
    pool = list(range(1, n * width + 2000))
    rng.shuffle(pool)
    tables = [[0] * width for _ in range(n + 3)]
    for s in slots:
        tables[s][:held[s]] = [pool.pop() for _ in range(held[s])]
    parent, start, q = [], [], []
    for b, s in enumerate(slots):
        fork = rng.random() < 0.8
        p = slots[(b + 1) % n] if seed == 0 else rng.choice(slots)           # (seed 0: everybody from its neighbour, in a circle)
        parent.append(p if fork and p != s else -1)
        start.append(rng.randint(0, held[p]) * PAGE if parent[-1] >= 0 else rng.randint((held[s] - 1) * PAGE + 1, held[s] * PAGE))
        q.append(rng.choice([0, 1, 3, 64, 200]))
    both(ops, start, q, slots, tables, pool, 2, width, sum(q) + 3, parent)


def test_a_fork_that_begins_inside_a_page_is_reported_and_gets_no_pages(ops):
    tables = [[0] * 3, [11, 12, 0], [0] * 3, [0] * 3]
    got = run_tables(ops, [100, 64, 70], [1, 1, 5], [1, 2, 3], tables, [31, 32, 33], 0, 3, 7, [-1, 1, 1])
    assert got[0] == [[11, 12, 0], [11, 31, 0], [0, 0, 0]]
    assert got[5] == [12 * PAGE + 36, 31 * PAGE] + [(70 + i) % PAGE for i in range(5)], "its tokens are on the reserved page"
    assert got[6] == [1] and got[7][3] == [0, 0, 0]
    with pytest.raises(ops.KernelError, match="inside a page"):
        ops.check_status()
    # a sequence that names its own record is none
    got = run_tables(ops, [70], [1], [1], tables, [31], 0, 3, 1, [1])
    assert got[0] == [[11, 12, 0]]
    ops.check_status()


def test_a_parent_outside_the_tables_is_reported(ops):
    got = run_tables(ops, [64], [1], [1], [[0] * 3, [11, 12, 0]], [31, 32, 33], 0, 3, 1, [5])
    assert got[0] == [[0, 0, 0]] and got[6] == [0]
    with pytest.raises(ops.KernelError, match="outside its tables"):
        ops.check_status()


def test_more_tokens_than_places_are_reported(ops):
    got = run_tables(ops, [0, 10], [3, 4], [1, 2], [[0] * 2, [0] * 2, [9, 0]], [31, 32], 0, 2, 5)
    assert got[3] == [0, 1, 2, 10, 11] and got[1] == [0, 3, 7]
    with pytest.raises(ops.KernelError, match="more tokens than places"):
        ops.check_status()
    run_tables(ops, [0, 10], [3, 4], [1, 2], [[0] * 2, [0] * 2, [9, 0]], [31, 32], 0, 2, 7)
    ops.check_status()
