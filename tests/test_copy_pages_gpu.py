"""Copies of whole cache pages against indexing; nothing but the named pages changes."""

from __future__ import annotations

import random

import pytest
import torch

import miniserve_b200  # noqa: F401
from miniserve_b200 import kernels
from miniserve_b200.kernels import KernelError

pytestmark = pytest.mark.gpu


def expected(pool, sources, destinations):
    want = pool.clone()
    for s, d in zip(sources, destinations):
        want[:, d] = pool[:, s]
    return want


def pools_of(shapes, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(shape, generator=g, device="cuda").to(dtype) for shape, dtype in shapes]


BF, F = torch.bfloat16, torch.float32


@pytest.mark.parametrize("shapes", [
    [((2, 40, 2, 16, 64), BF)] * 2,                                    # keys and values
    [((3, 40, 1, 1, 1), BF)],                                           # pages of two bytes
    [((3, 40, 3, 5, 25), F), ((3, 40, 3, 5, 7), F)],                    # pages of 1,500 and 420 bytes, heads of two sizes
    [((1, 40, 3, 1, 3), BF)],                                           # pages of 18 bytes
    [((5, 40, 24, 80), BF), ((1, 40, 16, 8, 128), F)],                  # latent vectors beside keys, other runs and types
    [((2, 40, 8, 128, 128), F)],                                        # half a megabyte to a page
    [((2, 40, 6), BF)] * 8,                                             # as many pools as a call takes
    [((1, 40, 40, 1024, 65), BF)],                                      # pages of 5 MB: more than the pieces of one round
])
@pytest.mark.parametrize("copies", [1, 7, 20])
def test_against_indexing(shapes, copies):
    order = list(range(40))
    random.Random(copies).shuffle(order)
    pools = pools_of(shapes)
    for sources in (order[20:20 + copies], [order[20]] * copies):
        want = [expected(p, sources, order[:copies]) for p in pools]
        kernels.copy_pages(pools, sources, order[:copies])
        for got, right in zip(pools, want):
            assert torch.equal(got, right)


@pytest.mark.parametrize("copies", [31, 32, 33, 899, 900, 901, 1999])
def test_many_pages(copies):
    pool = pools_of([((2, 4000, 2, 1, 4), BF)])[0]
    order = list(range(4000))
    random.Random(copies).shuffle(order)
    sources, destinations = order[:copies], order[copies:2 * copies]
    want = pool.clone()
    want[:, destinations] = pool[:, sources]
    kernels.copy_pages(pool, sources, destinations)
    assert torch.equal(pool, want)


def test_unaligned_pools():
    """A pool that starts two bytes behind a boundary, as a part of another tensor."""
    storage = torch.randn(1 + 2 * 10 * 64, device="cuda").to(BF)
    pool = storage[1:].view(2, 10, 64)
    want = expected(pool, [3, 4], [9, 0])
    kernels.copy_pages([pool], [3, 4], [9, 0])
    assert torch.equal(pool, want)


def test_offsets_pass_32_bits():
    pool = torch.empty((2, 70000, 8, 32, 128), dtype=BF, device="cuda")          # 9.2 GB
    pool[:, 5] = 3.0
    pool[:, 69999] = 1.0
    kernels.copy_pages([pool], [5], [69999])
    kernels.copy_pages([pool], [69999], [65537])
    assert (pool[:, 69999] == 3.0).all() and (pool[:, 65537] == 3.0).all()


def test_on_another_stream_and_captured():
    """In the order of the current stream; a captured call keeps its pages and copies what they hold at the replay."""
    pool = pools_of([((3, 12, 4, 16), F)])[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pool[:, 2] = 5.0
        kernels.copy_pages([pool], [2, 2], [7, 8])
        pool[:, 2] = 6.0
    stream.synchronize()
    assert (pool[:, 7] == 5.0).all() and (pool[:, 8] == 5.0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.copy_pages([pool], [2], [9])
    for value in (1.0, 2.0):
        pool[:, 2] = value
        graph.replay()
        torch.cuda.synchronize()
        assert (pool[:, 9] == value).all()


def test_refusals():
    pool = pools_of([((2, 10, 4, 8), BF)])[0]
    before = pool.clone()
    for pools, sources, destinations in (
            ([pool], [1], [1]), ([pool], [1, 2], [2, 3]), ([pool], [1, 2], [3, 3]), ([pool], [1], [10]), ([pool], [-1], [2]), ([pool], [1], [2, 3]),
            ([pool], [1.5], [2]), ([pool], [2 ** 40], [2]), ([pool], torch.tensor([1]), [2]), ([], [1], [2]), ([pool] * 9, [1], [2]),
            ([pool.cpu()], [1], [2]), ([pool.transpose(0, 1)], [1], [2]), ([pool[0]][:1] + [pool], [1], [2]), ([pool, pool[:, :5].contiguous()], [1], [2]),
            ([pool[:0]], [1], [2])):
        with pytest.raises(KernelError):
            kernels.copy_pages(pools, sources, destinations)
    kernels.copy_pages([pool], [], [])
    assert torch.equal(pool, before)
