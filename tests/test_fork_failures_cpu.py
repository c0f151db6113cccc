"""Forks and moves whose page copies fail: the cache is as it was before them."""

from __future__ import annotations

import copy
import gc
import weakref

import pytest

import miniserve_b200  # noqa: F401
from miniserve_b200.cache import CacheManager
from miniserve_b200.engine.step import StepFunction

from test_fork_cpu import FULL, OTHER, Pools


class Storage:
    """Copies on :class:`Pools`, or fails: before any copy, or after those of the first group."""

    def __init__(self, pools, after=None):
        self.pools, self.after = pools, after

    def copy_pages(self, copies):
        if self.after is not None:
            self.pools.copy([wanted if group < self.after else type(wanted)([], []) for group, wanted in enumerate(copies)])
            raise RuntimeError("no copy")
        self.pools.copy(copies)


def step_function(manager, storage):
    function = StepFunction.__new__(StepFunction)
    function.manager, function.storage = manager, storage
    return function


def held(manager):
    return ({name: (entry.length, copy.deepcopy(entry.tables)) for name, entry in manager.requests.items()},
            {digest: entry.pages for digest, entry in manager.prefix.entries.items()},
            [[allocator.refcount(page) for page in range(allocator.num_pages)] for allocator in manager.allocators],
            [allocator.free_count for allocator in manager.allocators])


@pytest.mark.parametrize("after", [0, 1])
def test_a_compaction_that_fails_changes_nothing(after):
    manager = CacheManager([FULL, OTHER], page_size=4, num_pages=40, max_seqs=6, enable_prefix_cache=True)
    pools = Pools(manager)
    for name, count in (("first", 30), ("p", 23), ("cached", 9)):
        manager.admit(name)
        pools.write(name, [f"{name}{i}" for i in range(count)])
    manager.cache_prefix("cached", list(range(9)))
    manager.release("cached")
    pools.copy(manager.fork("p", ["a", "b"]))
    manager.release("first")
    before, values = held(manager), {name: [pools.read(name, group) for group in range(2)] for name in manager.requests}
    changes = {name: entry.changes for name, entry in manager.requests.items()}
    with pytest.raises(RuntimeError, match="no copy"):
        step_function(manager, Storage(pools, after)).compact()
    assert held(manager) == before
    manager.check_invariants()
    assert {name: [pools.read(name, group) for group in range(2)] for name in manager.requests} == values
    # (whoever keeps a copy of a table has to look at it again)
    assert all(entry.changes > changes[name] for name, entry in manager.requests.items())
    step_function(manager, Storage(pools)).compact()          # and the same call can be made again
    assert held(manager) != before and all(allocator.refcount(page) for allocator in manager.allocators for page in range(allocator.used_count))
    manager.check_invariants()
    assert {name: [pools.read(name, group) for group in range(2)] for name in manager.requests} == values
    for name in list(manager.requests):
        pools.write(name, [1] * 7)
    manager.check_invariants()


@pytest.mark.parametrize("names", [lambda: ["a", "b"], lambda: iter(["a", "b"])], ids=["a list", "names that can be walked once"])
def test_a_fork_that_fails_changes_nothing(names):
    manager = CacheManager([FULL, OTHER], page_size=4, num_pages=20, max_seqs=4, enable_prefix_cache=True)
    pools = Pools(manager)
    manager.admit("p")
    pools.write("p", list(range(10)))
    before = held(manager)
    with pytest.raises(RuntimeError, match="no copy"):
        step_function(manager, Storage(pools, 1)).fork("p", names())
    assert held(manager) == before
    manager.check_invariants()
    step_function(manager, Storage(pools)).fork("p", names())
    assert all(pools.read(name, group) == list(range(10)) for name in "pab" for group in range(2))


def test_released_records_do_not_live_on_in_others():
    """A request that is kept while others come and go (a prompt that is forked) holds none of their records."""
    manager = CacheManager([FULL], page_size=4, num_pages=60, max_seqs=8)
    pools = Pools(manager)
    manager.admit("p")
    pools.write("p", list(range(12)))
    seen, live = [], ["p"]
    for i in range(20):                        # each new one stands behind the one before, as in the steps of a batch
        manager.fork("p", [f"r{i}"])
        live.append(f"r{i}")
        for name, other in zip(live[:-1], live[1:]):
            assert manager.shared_pages(name, other) == (3,)
        seen.append(weakref.ref(manager.requests[f"r{i}"]))
        if len(live) > 3:
            manager.release(live.pop(1))
        live = [name for name in live if name != "p"]          # (only the first time is it in a step)
    gc.collect()
    assert sum(record() is not None for record in seen) == len(manager.requests) - 1
    # the same name admitted again is another request
    manager.release("r19")
    manager.admit("r19")
    assert manager.shared_pages("r18", "r19") == (0,)
