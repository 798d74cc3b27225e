"""Sizes of the cache-budget workspaces, without a GPU."""
from __future__ import annotations

import pytest

from turboquant_amd import _lib


@pytest.mark.parametrize("budget", [70000, 1 << 20, 10 ** 9])
def test_evict_lists_are_bounded_by_the_table(budget):
    """256 rows of a table for 131072 tokens, 8 kv heads: no batch multiplies the
    budget.  Lists and keys take at most 4 bytes each per token and head."""
    room = 256 * 131072
    got = _lib.load().tq_evict_workspace_bytes(256, 8, room // 16, 16, budget)
    assert got <= 2 * room * 8 * 4 + 256 * 8 * 4 + 4096


def test_evict_lists_stay_small_under_small_budgets():
    """... nor the table the lists of a small budget."""
    room = 32 * 131072
    got = _lib.load().tq_evict_workspace_bytes(32, 8, room // 16, 16, 512)
    assert got <= 32 * 8 * 512 * 8 + room * 8 * 4 + 32 * 8 * 4 + 4096


def test_evict_workspace_grows_with_the_budget_up_to_the_table():
    lib, last = _lib.load(), 0
    for budget in (1, 100, 4096, 20000, 65536, 200000, 1 << 24):
        got = lib.tq_evict_workspace_bytes(64, 4, 64 * 8192, 16, budget)
        assert got >= last
        last = got
