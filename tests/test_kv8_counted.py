"""Counted page copies of the 8-bit cache: plan and count are read on the device, as the drafter's graphs use them."""

from __future__ import annotations

import pytest
import torch

from test_kv8 import Oracle, assert_pages, impl, make_cache, settle
from test_kv8_limits import ints, reported

PLAN = [(0, 4, 1), (0, 5, 16), (1, 6, 7), (7, 2, 3), (3, 8, 0)]


def copied(oracle, plan):
    for src, dst, n in plan:
        oracle.val[:, dst] = 0
        oracle.val[:, dst, :, :, :n] = oracle.val[:, src, :, :, :n]
        oracle.scale[:, dst] = oracle.scale[:, src] if n else 0


@pytest.mark.gpu
@pytest.mark.parametrize("count", [0, 1, 3, 5, 9, -1])
def test_counted_copies(count):
    """None, some and all rows of the plan; a count beyond the plan ends at its last row, a negative one copies none."""
    ops = impl("cuda")
    cache = make_cache("cuda", 3, 10, 2, 16, 128, seed=count + 2, empty=(7,))
    oracle = Oracle(cache)
    copied(oracle, PLAN[: max(0, count)])
    ops.kv8_copy_pages_counted(cache, ints(PLAN, "cuda"), ints([count, 77], "cuda"))
    settle(ops)
    assert_pages(cache, oracle)


@pytest.mark.gpu
def test_rows_behind_the_count_are_not_looked_at():
    """A plan's unused rows may hold anything, also what would be refused or clash with a used row."""
    ops = impl("cuda")
    cache = make_cache("cuda", 2, 10, 1, 16, 128, seed=0)
    oracle = Oracle(cache)
    copied(oracle, PLAN[:2])
    ops.kv8_copy_pages_counted(cache, ints([*PLAN[:2], (4, 0, 3), (99, -5, 40), (1, 4, 2)], "cuda"), ints([2], "cuda"))
    settle(ops)
    assert_pages(cache, oracle)
    before = Oracle(cache)
    reported("cuda", lambda o: o.kv8_copy_pages_counted(cache, ints([(1, 10, 2), (2, 3, 1)], "cuda"), ints([1], "cuda")), 2)
    assert_pages(cache, before)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 64, 200])
def test_a_captured_copy_follows_its_plan_and_count(rows):
    """One graph, replayed over plans of different lengths."""
    ops = impl("cuda")
    cache = make_cache("cuda", 2, 2 * rows + 2, 2, 16, 128, seed=rows)
    oracle = Oracle(cache)
    plan, count = torch.zeros(rows, 3, dtype=torch.int32, device="cuda"), ints([0], "cuda")
    ops.kv8_copy_pages_counted(cache, plan, count)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv8_copy_pages_counted(cache, plan, count)
    g = torch.Generator().manual_seed(rows)
    for n in (rows, 0, -(-rows // 2), 1):
        perm = torch.randperm(2 * rows + 2, generator=g).tolist()
        now = [(perm[rows + i], perm[i], int(torch.randint(0, 17, (1,), generator=g))) for i in range(n)]
        copied(oracle, now)
        if n:
            plan[:n] = ints(now, "cuda")
        count.fill_(n)
        graph.replay()
        settle(ops)
        assert_pages(cache, oracle)
