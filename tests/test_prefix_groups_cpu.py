"""How a step's requests are cut into groups that share a prefix, on the CPU."""

from __future__ import annotations

import random

import pytest

import miniserve_b200  # noqa: F401
from miniserve_b200.cache import CacheManager
from miniserve_b200.engine.step import SHARED_KEYS_LEAST, StepFunction
from miniserve_b200.parts import CacheGroup, PagedKVNeed


def grouped(tables, least=1, page_size=16):
    """The groups that requests with these block tables (whole pages) form."""
    manager = CacheManager([CacheGroup(PagedKVNeed(2, 16, None), 1)], page_size, 5000, 64)
    for name, table in enumerate(tables):
        entry = manager.admit(str(name))
        entry.tables, entry.length = [list(table)], len(table) * page_size
    function = StepFunction.__new__(StepFunction)
    function.manager = manager
    return function._shared_groups([str(i) for i in range(len(tables))], 0, least)


def saved(groups):
    return sum((count - 1) * keys for count, keys in groups)


def every_cut(n):
    for cuts in range(2 ** (n - 1)):
        starts = [0] + [i + 1 for i in range(n - 1) if cuts >> i & 1] + [n]
        yield list(zip(starts[:-1], starts[1:]))


SYSTEM, DOCUMENT, OTHER = list(range(8)), list(range(100, 1092)), list(range(2000, 2040))


@pytest.mark.parametrize("order", ["the short one first", "the short one last", "the short one between"])
def test_a_short_common_start_beside_a_long_one(order):
    """One request that shares 128 keys with its neighbours does not cost them their 16,000."""
    long = [SYSTEM + DOCUMENT + [3000 + i] for i in range(5)]
    short = [SYSTEM + [4000]]
    tables = {"the short one first": short + long, "the short one last": long + short, "the short one between": long[:2] + short + long[2:]}[order]
    groups = grouped(tables)
    want = {"the short one first": [(1, 0), (5, 16000)], "the short one last": [(5, 16000), (1, 0)],
            "the short one between": [(2, 16000), (1, 0), (3, 16000)]}[order]
    assert sorted(groups) == sorted(want) and saved(groups) == saved(want)


def test_two_documents_behind_one_system_prompt():
    tables = [SYSTEM + DOCUMENT + [3000 + i] for i in range(3)] + [SYSTEM + OTHER + [3100 + i] for i in range(4)] + [SYSTEM + [3200 + i] for i in range(3)]
    assert grouped(tables) == [(3, 16000), (4, 768), (3, 128)]


def test_few_keys_are_no_group():
    few, enough = SYSTEM[:7], SYSTEM
    assert grouped([few + [3000 + i] for i in range(9)]) is None
    assert grouped([enough + [3000 + i] for i in range(9)]) == [(9, 128)]
    assert grouped([enough + [3000 + i] for i in range(9)], least=8 * 128 + 1) is None
    assert grouped([[1, 2], [3]]) is None and grouped([SYSTEM]) is None


@pytest.mark.parametrize("seed", range(8))
def test_no_cut_saves_more(seed):
    rng = random.Random(seed)
    for _ in range(12):
        n, tables, next_page = rng.randint(1, 9), [], 0
        for _ in range(n):
            keep = rng.choice([0, 2, 8, 8, 9, 12, 30, 200]) if tables else 0
            fresh = rng.choice([1, 3, 9, 40, 200])
            tables.append((tables[-1][:keep] if tables else []) + list(range(next_page, next_page + fresh)))
            next_page += fresh
        def shares(first, end):
            alike = 0
            while all(len(t) > alike and t[alike] == tables[first][alike] for t in tables[first:end]):
                alike += 1
            return 16 * alike if end - first > 1 and 16 * alike >= SHARED_KEYS_LEAST else 0
        best = max(sum((end - first - 1) * shares(first, end) for first, end in cut) for cut in every_cut(n))
        groups = grouped(tables)
        if best == 0:
            assert groups is None
            continue
        assert sum(count for count, _ in groups) == n and saved(groups) == best
        first = 0
        for count, keys in groups:                     # what is said to be shared is
            assert keys == shares(first, first + count)
            first += count
