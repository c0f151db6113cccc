"""Forks and moves of a paged cache on the CPU: what every request reads through its table stays what it wrote, whatever is shared, copied or moved."""

from __future__ import annotations

import random

import pytest

import miniserve_b200  # noqa: F401
from miniserve_b200.cache import CacheManager, OutOfPagesError, OutOfSlotsError, PageAllocator
from miniserve_b200.parts import CacheGroup, PagedKVNeed, StateNeed

FULL, OTHER = CacheGroup(PagedKVNeed(2, 16, None), 3), CacheGroup(PagedKVNeed(1, 8, None), 1)


class Pools:
    """What a device would hold: per group, a value for every slot."""

    def __init__(self, manager):
        self.manager, self.pools = manager, [dict() for _ in manager.allocators]

    def write(self, request_id, values):
        reservation = self.manager.prepare([(request_id, len(values))])
        for pool, slots in zip(self.pools, reservation.items[0].slots):
            for slot, value in zip(slots, values):
                pool[int(slot)] = value
        self.manager.commit(reservation)

    def copy(self, copies):
        size = self.manager.page_size
        for pool, wanted in zip(self.pools, copies):
            assert len(set(wanted.destinations)) == len(wanted.destinations) and not set(wanted.destinations) & set(wanted.sources)
            for source, destination in zip(wanted.sources, wanted.destinations):
                for offset in range(size):
                    pool[destination * size + offset] = pool.get(source * size + offset)

    def read(self, request_id, group):
        entry, size = self.manager.requests[request_id], self.manager.page_size
        return [self.pools[group][entry.tables[group][i // size] * size + i % size] for i in range(entry.length)]


def test_allocator_compacts():
    allocator = PageAllocator(8)
    allocator.allocate(7)
    for page in (0, 2, 3):
        allocator.release(page)
    allocator.retain(6)
    assert allocator.compact() == {6: 0, 5: 2, 4: 3}
    assert [allocator.refcount(p) for p in range(8)] == [2, 1, 1, 1, 0, 0, 0, 0]
    allocator.check_invariants()
    assert allocator.compact() == {} and allocator.allocate(2) == [4, 5]
    assert PageAllocator(3).compact() == {}


@pytest.mark.parametrize("length", [0, 1, 3, 4, 5, 8, 11])
def test_a_fork_shares_full_pages_and_copies_the_last(length):
    manager = CacheManager([FULL, OTHER], page_size=4, num_pages=20, max_seqs=4)
    pools = Pools(manager)
    manager.admit("p")
    if length:
        pools.write("p", list(range(length)))
    copies = manager.fork("p", ["a", "b"])
    pools.copy(copies)
    manager.check_invariants()
    for group in range(2):
        assert len(copies[group].sources) == (2 if length % 4 else 0)
        for child in ("a", "b"):
            assert manager.requests[child].tables[group][:length // 4] == manager.requests["p"].tables[group][:length // 4]
            assert pools.read(child, group) == list(range(length))
    # each writes on in its own page
    for name in ("p", "a", "b"):
        pools.write(name, [f"{name}{i}" for i in range(6)])
    for name in ("p", "a", "b"):
        for group in range(2):
            assert pools.read(name, group) == list(range(length)) + [f"{name}{i}" for i in range(6)]
    manager.release("p")
    manager.truncate("a", length // 4 * 4)
    manager.release("b")
    manager.release("a")
    manager.check_invariants()
    assert all(a.free_count == 20 for a in manager.allocators)


def test_a_fork_that_does_not_fit_changes_nothing():
    manager = CacheManager([FULL], page_size=4, num_pages=3, max_seqs=8)
    pools = Pools(manager)
    manager.admit("p")
    pools.write("p", list(range(6)))
    with pytest.raises(OutOfPagesError):
        manager.fork("p", ["a", "b"])
    assert set(manager.requests) == {"p"} and manager.allocators[0].free_count == 1
    manager.check_invariants()
    few = CacheManager([FULL], page_size=4, num_pages=30, max_seqs=2)
    few.admit("p")
    with pytest.raises(OutOfSlotsError):
        few.fork("p", ["a", "b"])
    for wrong in (["p"], ["a", "a"]):
        with pytest.raises(RuntimeError):
            manager.fork("p", wrong)
    reservation = manager.prepare([("p", 1)])
    for refused in (lambda: manager.fork("p", ["a"]), manager.compact):
        with pytest.raises(RuntimeError):
            refused()
    manager.abort(reservation)
    with pytest.raises(KeyError):
        manager.fork("nobody", ["a"])
    assert manager.fork("p", []) [0].sources == []
    manager.check_invariants()


def test_windows_and_states_are_refused():
    for groups in ([CacheGroup(PagedKVNeed(2, 16, 8), 1)], [FULL, CacheGroup(StateNeed((4,)), 1)]):
        manager = CacheManager(groups, 4, 8, 4)
        manager.admit("p")
        with pytest.raises(RuntimeError):
            manager.fork("p", ["a"])


def test_a_fork_evicts_cached_prefixes_when_it_needs_their_pages():
    manager = CacheManager([FULL], page_size=4, num_pages=4, max_seqs=4, enable_prefix_cache=True)
    pools = Pools(manager)
    manager.admit("old")
    pools.write("old", list(range(8)))
    manager.cache_prefix("old", list(range(8)))
    manager.release("old")
    manager.admit("p")
    pools.write("p", [50, 51])
    pools.copy(manager.fork("p", ["a", "b", "c"]))
    manager.check_invariants()
    assert [pools.read(n, 0) for n in "pabc"] == [[50, 51]] * 4


@pytest.mark.parametrize("seed", range(6))
def test_random_orders(seed):
    rng = random.Random(seed)
    manager = CacheManager([FULL, OTHER], page_size=4, num_pages=60, max_seqs=10, enable_prefix_cache=True, prefix_cache_max_entries=8)
    pools, live, counter = Pools(manager), {}, 0
    for _ in range(300):
        choice = rng.random()
        try:
            if choice < 0.15 and manager.slots.free_count:
                name = f"r{counter}"
                counter += 1
                prompt = [rng.randrange(3) for _ in range(rng.randint(1, 14))]
                manager.admit(name)
                matched = manager.attach_prefix(name, prompt)
                live[name] = prompt[:matched]
                pools.write(name, prompt[matched:])
                live[name] = list(prompt)
                if rng.random() < 0.5:
                    manager.cache_prefix(name, prompt)
            elif choice < 0.35 and live:
                parent = rng.choice(sorted(live))
                names = [f"r{counter + i}" for i in range(rng.randint(1, 3))]
                pools.copy(manager.fork(parent, names))
                counter += len(names)
                live.update({name: list(live[parent]) for name in names})
            elif choice < 0.65 and live:
                name = rng.choice(sorted(live))
                values = [rng.randrange(3, 1000) for _ in range(rng.randint(1, 6))]
                pools.write(name, values)
                live[name] += values
            elif choice < 0.75 and live:
                name = rng.choice(sorted(live))
                length = rng.randint(0, len(live[name])) // 4 * 4
                manager.truncate(name, length)
                del live[name][length:]
            elif choice < 0.85:
                pools.copy(manager.compact())
                for allocator in manager.allocators:
                    assert all(allocator.refcount(p) > 0 for p in range(allocator.used_count))
            elif live:
                name = rng.choice(sorted(live))
                manager.release(name)
                del live[name]
        except (OutOfPagesError, OutOfSlotsError):
            for name in [n for n in manager.requests if n not in live or len(live[n]) != manager.length(n)]:
                manager.release(name)
                live.pop(name, None)
        manager.check_invariants()
        for name, values in live.items():
            for group in range(2):
                assert pools.read(name, group) == values
