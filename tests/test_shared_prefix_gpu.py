"""Attention of a batch whose requests share a prefix against attention in float64, request by request.

The bounds are worked out from the number formats.  With w_t a row's softmax weights, A = sum_t w_t |v_t| and o the exact output: every weight may be
rounded to the type's half step h before it multiplies a value (h A), the output is rounded once (h |o|), and the float32 arithmetic of
scores, exponents and sums moves every weight by a relative ``_float_part`` (see there) that A is multiplied with."""

from __future__ import annotations

import math

import pytest
import torch

import miniserve_b200  # noqa: F401
from miniserve_b200 import kernels
from miniserve_b200.kernels import KernelError

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def make(groups, prefix, queries, suffix, heads=8, kv_heads=2, d=64, page=16, dtype=torch.bfloat16, seed=0, sink=None, softcap=None,
         stale=float("nan"), peak=1.5):
    """A step: ``groups`` requests to a group, their prefixes, new tokens and keys behind the prefix (the new ones included).  Pages lie in no order; what
    belongs to no context is ``stale``."""
    g = torch.Generator().manual_seed(seed)
    of_request = [i for i, count in enumerate(groups) for _ in range(count)]
    context = [prefix[of_request[r]] + suffix[r] for r in range(len(queries))]
    shared = [p // page for p in prefix]
    needed = [(c + page - 1) // page for c in context]
    total = sum(shared) + sum(n - shared[of_request[r]] for r, n in enumerate(needed)) + 2
    order = torch.randperm(total, generator=g).tolist()
    k_pool = torch.full((total, kv_heads, page, d), stale)
    v_pool = torch.full((total, kv_heads, page, d), stale)
    at, group_pages = 0, []
    for count in shared:
        group_pages.append(order[at:at + count])
        at += count
    width, tables, filled = max(needed + [1]), [], set()
    for r, n in enumerate(needed):
        pages = group_pages[of_request[r]] + order[at:at + n - shared[of_request[r]]]
        at += n - shared[of_request[r]]
        tables.append(pages + [total - 1] * (width - n))
        for index, page_number in enumerate(pages):
            live = min(page, context[r] - index * page)
            if (page_number, live) not in filled:
                filled.add((page_number, live))
                k_pool[page_number, :, :live] = torch.randn(kv_heads, live, d, generator=g)
                v_pool[page_number, :, :live] = torch.randn(kv_heads, live, d, generator=g)
        # (a page that a prefix ends in is a copy for each of its requests but the first: the prefix's keys in it are the same)
        own = prefix[of_request[r]] % page
        first = of_request.index(of_request[r])
        if own and r != first:
            for pool in (k_pool, v_pool):
                pool[pages[shared[of_request[r]]], :, :own] = pool[tables[first][shared[of_request[r]]], :, :own]
    starts = [0]
    for count in queries:
        starts.append(starts[-1] + count)
    group_start = [0]
    for count in groups:
        group_start.append(group_start[-1] + count)
    positions = [context[r] - queries[r] + i for r in range(len(queries)) for i in range(queries[r])]
    ints = lambda values: torch.tensor(values, dtype=torch.int32).cuda()
    tokens = [starts[b] - starts[a] for a, b in zip(group_start[:-1], group_start[1:])]
    scores = torch.randn(heads, generator=g).cuda() if sink == "scores" else bool(sink)
    return dict(q=(peak * torch.randn(starts[-1], heads, d, generator=g)).to(dtype).cuda(), k_pool=k_pool.to(dtype).cuda(), v_pool=v_pool.to(dtype).cuda(),
                block_tables=ints(tables).view(len(tables), width), positions=ints(positions), query_start=ints(starts), context_lens=ints(context),
                group_start=ints(group_start), prefix_lens=ints(prefix), max_query_len=max(queries), max_group_tokens=max(tokens),
                max_prefix_len=max(prefix), max_suffix_len=max(suffix), scale=d ** -0.5, softcap=softcap, sink=scores)


def attend(step, out=None, **other):
    out = torch.full_like(step["q"], float("nan")) if out is None else out
    kernels.shared_prefix_attention(out=out, **{**step, **other})
    return out


def _float_part(d, keys, largest, softcap):
    """A score is a sum of d products in float32, scaled (and capped): off by at most (d + 4) 2^-24 sum |q k| scale; the exponential of it, its running
    maximum and the correction of older terms add a few 2^-22; a sum of n terms is off by n 2^-24, in the joins of at most 128 parts too."""
    score = (d + 4) * 2.0 ** -24 * largest + (2.0 ** -21 * softcap if softcap else 0.0) + 2.0 ** -22 * largest
    return 2.0 * score + 16 * 2.0 ** -22 + (keys + 160) * 2.0 ** -24


def expected(step):
    """(output, bound of the error) in float64."""
    q, tables, starts = step["q"].double(), step["block_tables"].tolist(), step["query_start"].tolist()
    page, n_kv = step["k_pool"].shape[2], step["k_pool"].shape[1]
    n, n_q, d = q.shape
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    h = HALF_STEP[step["q"].dtype]
    for r, length in enumerate(step["context_lens"].tolist()):
        if starts[r] == starts[r + 1]:
            continue
        pages = torch.tensor(tables[r][:(length + page - 1) // page], device=q.device)
        keys, values = (pool[pages].transpose(1, 2).reshape(-1, n_kv, d)[:length].double().repeat_interleave(n_q // n_kv, 1)
                        for pool in (step["k_pool"], step["v_pool"]))
        for token in range(starts[r], starts[r + 1]):
            last = int(step["positions"][token]) + 1
            products = torch.einsum("hd,khd->hk", q[token], keys[:last]) * step["scale"]
            absolute_products = torch.einsum("hd,khd->hk", q[token].abs(), keys[:last].abs()) * step["scale"]
            if step["softcap"]:
                products = step["softcap"] * torch.tanh(products / step["softcap"])
            if step["sink"] is not False:
                sink = step["sink"].double() if isinstance(step["sink"], torch.Tensor) else torch.zeros(n_q, device=q.device, dtype=torch.float64)
                products = torch.cat([products, sink[:, None]], 1)
            weights = torch.softmax(products, -1)[:, :last]
            largest = float(absolute_products[weights > 0.0].max())          # (a key without weight is far from having any)
            out[token] = torch.einsum("hk,khd->hd", weights, values[:last])
            absolute = torch.einsum("hk,khd->hd", weights, values[:last].abs())
            bound[token] = h * (absolute + out[token].abs()) + _float_part(d, last, largest, step["softcap"]) * absolute + 1e-30
    return out, bound


def check(step, got):
    want, bound = expected(step)
    finite, worst = bool(torch.isfinite(got).all()), float(((got.double() - want).abs() / bound).max())
    assert finite and worst <= 1.0, f"error is {worst:.3f} of its bound"


CASES = {
    "one request, one key": dict(groups=[1], prefix=[0], queries=[1], suffix=[1]),
    "one request, all of it a prefix but its token": dict(groups=[1], prefix=[160], queries=[1], suffix=[1]),
    "two samples": dict(groups=[2], prefix=[512], queries=[1, 1], suffix=[17, 5], heads=16, kv_heads=8, d=128),
    "a prefix that ends inside a tile": dict(groups=[5], prefix=[144], queries=[1] * 5, suffix=[1, 2, 3, 200, 31], d=128),
    "a prefix that ends inside a page": dict(groups=[3], prefix=[131], queries=[1, 2, 1], suffix=[1, 2, 60], d=128),
    "prefix of one key": dict(groups=[4], prefix=[1], queries=[1] * 4, suffix=[1, 5, 9, 64], page=1, d=64),
    "groups of every kind": dict(groups=[3, 1, 6, 1], prefix=[272, 0, 1040, 64], queries=[1, 2, 1, 5, 1, 1, 3, 1, 1, 1, 4],
                                 suffix=[5, 2, 1, 90, 33, 1, 3, 700, 12, 1, 4], d=64),
    "a request without tokens": dict(groups=[3, 2], prefix=[96, 48], queries=[1, 0, 2, 0, 1], suffix=[4, 3, 2, 1, 7]),
    "long portions behind a prefix": dict(groups=[2, 2], prefix=[320, 0], queries=[70, 1, 33, 129], suffix=[70, 3, 40, 129], d=128),
    "long prefix, many parts": dict(groups=[3], prefix=[9008], queries=[1, 1, 1], suffix=[16, 3, 2000], heads=8, kv_heads=1, d=128),
    "more rows than a tile": dict(groups=[40], prefix=[400], queries=[1] * 40, suffix=[1 + 7 * i for i in range(40)], heads=32, kv_heads=4, d=128),
    "three heads to a key head": dict(groups=[50, 2], prefix=[256, 96], queries=[1] * 52, suffix=[3] * 52, heads=6, kv_heads=2, d=64),
    "five heads to a key head": dict(groups=[30], prefix=[384], queries=[2] * 30, suffix=[9] * 30, heads=5, kv_heads=1, d=128),
    "twenty heads to a key head": dict(groups=[4], prefix=[200], queries=[1, 3, 1, 2], suffix=[9, 3, 1, 50], heads=40, kv_heads=2, d=64, page=8),
    "as many key heads as heads": dict(groups=[9], prefix=[128], queries=[1] * 9, suffix=[130] * 9, heads=4, kv_heads=4, d=128),
    "pages of 24": dict(groups=[6], prefix=[600], queries=[1, 1, 2, 1, 1, 1], suffix=[25, 1, 2, 3, 100, 24], page=24, d=128),
    "pages of 128": dict(groups=[6], prefix=[640], queries=[1] * 6, suffix=[128, 1, 129, 3, 300, 24], page=128, d=64),
    "pages of 100": dict(groups=[6], prefix=[700], queries=[1] * 6, suffix=[128, 1, 129, 3, 300, 24], page=100, d=128),
    "head size 40": dict(groups=[4, 3], prefix=[272, 80], queries=[1, 2, 1, 1, 1, 1, 3], suffix=[5, 20, 1, 90, 33, 1, 3], d=40),
    "head size 80": dict(groups=[4], prefix=[272], queries=[1] * 4, suffix=[5, 20, 1, 90], d=80),
    "head size 7": dict(groups=[4], prefix=[272], queries=[1] * 4, suffix=[5, 20, 1, 90], d=7),
    "head size 256": dict(groups=[4], prefix=[96], queries=[1, 1, 2, 1], suffix=[5, 20, 2, 90], d=256),
    "head size 512": dict(groups=[4], prefix=[96], queries=[1, 1, 2, 1], suffix=[5, 20, 2, 90], d=512),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("name", sorted(CASES))
def test_against_float64(name, dtype):
    """Pages behind a context and pages of nobody are NaN throughout."""
    step = make(dtype=dtype, **CASES[name])
    check(step, attend(step))


@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("sink,softcap", [(True, None), ("scores", None), (False, 5.0), ("scores", 30.0)])
def test_sinks_and_soft_caps(dtype, d, sink, softcap):
    step = make(groups=[6, 2], prefix=[208, 0], queries=[1, 3, 1, 1, 2, 1, 1, 4], suffix=[1, 9, 33, 150, 2, 64, 1, 40], d=d, dtype=dtype, sink=sink,
                softcap=softcap)
    check(step, attend(step))


@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
def test_scores_of_every_size(dtype, d):
    """Scores up to some hundreds: the running maximum grows and falls over the keys, most weights vanish."""
    step = make(groups=[7], prefix=[1500], queries=[1] * 7, suffix=[3, 300, 1, 64, 65, 2, 31], d=d, dtype=dtype, peak=40.0, page=20)
    check(step, attend(step))


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.bfloat16, 40), (torch.float32, 64)])
def test_infinite_and_lowest_keys(dtype, d):
    """Keys that no row gives any weight: one of the prefix is minus infinity throughout, one of a request's own holds the type's lowest numbers, and
    the queries are positive."""
    step = make(groups=[4], prefix=[160], queries=[1] * 4, suffix=[5, 1, 70, 33], d=d, dtype=dtype, heads=4, kv_heads=1)
    step["q"].abs_()
    step["k_pool"][step["block_tables"][0, 3].long(), :, 5] = -float("inf")
    step["k_pool"][step["block_tables"][2, -1].long(), :, 0] = torch.finfo(dtype).min
    got = attend(step)
    check(step, got)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 48), (torch.float32, 64)])
def test_same_as_without_sharing(dtype, d):
    """Every request a group of its own with no prefix, and all behind one: the same within both bounds."""
    step = make(groups=[8], prefix=[336], queries=[1, 2, 1, 1, 3, 1, 1, 1], suffix=[20, 2, 1, 9, 3, 100, 64, 17], d=d, dtype=dtype)
    n = step["context_lens"].numel()
    ints = lambda values: torch.tensor(values, dtype=torch.int32).cuda()
    alone = {**step, "group_start": ints(list(range(n + 1))), "prefix_lens": ints([0] * n), "max_prefix_len": 0, "max_suffix_len": 336 + 100,
             "max_group_tokens": 3}
    check(step, attend(step))
    check(step, attend(alone))
    check(step, attend({**alone, "max_prefix_len": 500, "max_group_tokens": 30}))          # (bounds are upper bounds)


def test_against_paged_attention():
    step = make(groups=[6], prefix=[512], queries=[1, 2, 1, 1, 5, 1], suffix=[20, 2, 1, 9, 5, 100], d=128, heads=16, kv_heads=8)
    requests = torch.repeat_interleave(torch.arange(6, device="cuda"), step["query_start"].diff()).int()
    out = torch.empty_like(step["q"])
    finite = lambda pool: torch.nan_to_num(pool, nan=0.0)
    kernels.paged_attention(step["q"], finite(step["k_pool"]), finite(step["v_pool"]), step["block_tables"], requests, step["positions"],
                            step["query_start"], step["context_lens"], 5, 612, step["scale"], None, out)
    check(step, out)
    check(step, attend(step))


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 40), (torch.float32, 64)])
def test_rows_behind_the_last_request_stay(dtype, d):
    """Padding behind the last request (in q and out) is left alone, and the same call gives the same bits."""
    step = make(groups=[5], prefix=[160], queries=[1, 2, 1, 1, 3], suffix=[20, 2, 1, 9, 3], d=d, dtype=dtype)
    first = attend(step)
    n = first.shape[0]
    padded = {**step, "q": torch.cat([step["q"], torch.full_like(step["q"][:3], float("nan"))]),
              "positions": torch.cat([step["positions"], torch.zeros(3, dtype=torch.int32, device="cuda")])}
    out = torch.full_like(padded["q"], 7.0)
    attend(padded, out)
    assert torch.equal(out[:n], first) and (out[n:] == 7.0).all()
    assert torch.equal(attend(step), first)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 48), (torch.float32, 64)])
def test_captured_with_growing_contexts(dtype, d):
    """A captured call whose lengths, tables and prefixes change between replays, two graphs in turn, and on a stream of its own."""
    steps = [make(groups=[4, 2], prefix=[p, 48], queries=[1] * 6, suffix=[s, 1, 2, 3, s + 5, 9], d=d, dtype=dtype, seed=s) for p, s in ((240, 3), (160, 40), (0, 7))]
    width, pages = max(s["block_tables"].shape[1] for s in steps), max(s["k_pool"].shape[0] for s in steps)
    for s in steps:
        s["block_tables"] = torch.nn.functional.pad(s["block_tables"], (0, width - s["block_tables"].shape[1]))
        for name in ("k_pool", "v_pool"):
            s[name] = torch.cat([s[name], torch.full((pages - s[name].shape[0],) + s[name].shape[1:], float("nan"), dtype=dtype, device="cuda")])
    bounds = dict(max_query_len=1, max_group_tokens=4, max_prefix_len=256, max_suffix_len=64)
    tensors = [k for k, v in steps[0].items() if isinstance(v, torch.Tensor)]
    held = [{k: (v.clone() if k in tensors else v) for k, v in {**steps[0], **bounds}.items()} for _ in range(2)]
    outs = [torch.empty_like(steps[0]["q"]) for _ in range(2)]
    graphs = []
    attend(held[0], outs[0])
    torch.cuda.synchronize()
    for step, out in zip(held, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(step, out)
        graphs.append(graph)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for first, second in ((0, 1), (1, 2), (2, 0)):
            for which, at in ((0, first), (1, second)):
                for k in tensors:
                    held[which][k].copy_(steps[at][k])
                outs[which].fill_(float("nan"))
                graphs[which].replay()
            stream.synchronize()
            for which, at in ((0, first), (1, second)):
                check(steps[at], outs[which])


def test_long_cache_offsets_pass_32_bits():
    """A pool of more than 2^32 bytes and 2^31 entries: the last pages hold the keys."""
    pages, kv_heads, page, d = 66000, 8, 32, 128
    step = make(groups=[3], prefix=[320], queries=[1, 1, 2], suffix=[40, 1, 2], heads=16, kv_heads=kv_heads, d=d, page=page)
    used = step["k_pool"].shape[0]
    for name in ("k_pool", "v_pool"):
        big = torch.empty((pages, kv_heads, page, d), dtype=torch.bfloat16, device="cuda")
        big[pages - used:] = step[name]
        step[name + "_small"], step[name] = step[name], big
    small = {**step, "k_pool": step.pop("k_pool_small"), "v_pool": step.pop("v_pool_small")}
    small.pop("k_pool_small", None), small.pop("v_pool_small", None)
    got = attend({**step, "block_tables": step["block_tables"] + (pages - used)})
    check(small, got)


@pytest.mark.parametrize("dtype,d,page", [(torch.bfloat16, 128, 16), (torch.bfloat16, 64, 5), (torch.bfloat16, 48, 16), (torch.float32, 64, 16)])
@pytest.mark.parametrize("count", [2, 12])
def test_table_entries_behind_a_context_are_not_read(dtype, d, page, count):
    """Entries behind a request's last page hold no page numbers at all."""
    step = make(groups=[count, 1], prefix=[7 * page, 0], queries=[1] * (count + 1), suffix=[1 + 9 * i for i in range(count + 1)], d=d, dtype=dtype, page=page)
    table, rows = step["block_tables"], step["context_lens"].tolist()
    for r, length in enumerate(rows):
        table[r, (length + page - 1) // page:] = (-1, 2 ** 31 - 1, 10 ** 6)[r % 3]
    check(step, attend(step))


@pytest.mark.parametrize("dtype,d,page", [(torch.bfloat16, 128, 16), (torch.bfloat16, 64, 5), (torch.bfloat16, 48, 16), (torch.float32, 64, 16)])
def test_nan_stays_with_its_request(dtype, d, page):
    """NaN among a request's own keys makes its outputs NaN, and nobody else's."""
    step = make(groups=[20], prefix=[10 * page], queries=[1] * 20, suffix=[page + 3] * 20, d=d, dtype=dtype, page=page)
    step["k_pool"][step["block_tables"][4, 10].long(), :, 2] = float("nan")
    got = attend(step)
    assert torch.isnan(got[4]).all()
    others = [r for r in range(20) if r != 4]
    want, bound = expected({**step, "k_pool": torch.nan_to_num(step["k_pool"], nan=0.0)})
    assert ((got.double() - want).abs()[others] <= bound[others]).all()


def test_refusals():
    step = make(groups=[2], prefix=[32], queries=[1, 1], suffix=[3, 4])
    bad = [dict(q=step["q"].cpu()), dict(q=step["q"].half()), dict(k_pool=step["k_pool"].float()), dict(v_pool=step["v_pool"][:, :, :8]),
           dict(q=step["q"].transpose(0, 1)), dict(q=step["q"][:, :5].contiguous()), dict(positions=step["positions"].long()),
           dict(block_tables=step["block_tables"][:1]), dict(query_start=step["query_start"][:2]), dict(context_lens=step["context_lens"].cpu()),
           dict(group_start=step["group_start"][:1]), dict(prefix_lens=step["prefix_lens"].float()), dict(max_query_len=-1), dict(max_prefix_len=-1),
           dict(max_group_tokens=0), dict(softcap=-1.0), dict(softcap=float("nan")), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(sink=torch.zeros(3, device="cuda")),
           dict(group_start=step["group_start"][:1], prefix_lens=step["prefix_lens"][:0])]
    for other in bad:
        with pytest.raises(KernelError):
            attend(step, out=torch.empty_like(step["q"]), **other)
    with pytest.raises(KernelError):
        attend(step, out=torch.empty_like(step["q"][:1]))
    none = {k: (v[:0] if k in ("q", "positions") else v) for k, v in step.items()}
    assert attend(none).shape[0] == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", [dict(groups=[6], prefix=[600], queries=[1, 1, 2, 1, 1, 1], suffix=[25, 1, 2, 3, 100, 24], page=24),
                                  dict(groups=[6], prefix=[2016], queries=[2] * 6, suffix=[5, 2, 9, 64, 3, 17]),
                                  dict(groups=[60, 2], prefix=[264, 96], queries=[1] * 62, suffix=[3] * 62, heads=6, kv_heads=2, page=24)],
                         ids=["pages of 24", "a prefix that ends inside a tile", "rows that no token fills"])
def test_capped_bits_do_not_depend_on_earlier_work(case, d):
    """The same call after calls that leave small and large numbers in shared memory, where keys behind a prefix and rows without a token are never loaded:
    the same bits.  The cap is high, so that another way of rounding a score shows in the result."""
    step, earlier = make(d=d, softcap=1000.0, **case), make(groups=[64], prefix=[8192], queries=[1] * 64, suffix=[1] * 64, d=d)
    got = []
    for left in (0.0, 3e4, -3e4, 0.0):
        attend({**earlier, **{name: torch.full_like(earlier[name], left) for name in ("q", "k_pool", "v_pool")}})
        got.append(attend(step))
    assert all(torch.equal(other, got[0]) for other in got[1:])
    check(step, got[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
def test_an_infinite_cap_is_refused(dtype):
    """(It would multiply by infinity what tanh gave; no cap is None or 0.)"""
    step = make(groups=[2], prefix=[32], queries=[1, 1], suffix=[3, 4], dtype=dtype)
    with pytest.raises(KernelError):
        attend(step, softcap=float("inf"))
    check(step, attend(step, softcap=0.0))


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 40), (torch.float32, 64)])
def test_a_batch_without_any_token(dtype, d):
    """Rows of padding alone, whose bounds say that no request brings a token: nothing is computed and nothing written."""
    step = make(groups=[2, 1], prefix=[32, 0], queries=[0, 0, 0], suffix=[3, 4, 1], d=d, dtype=dtype)
    step["q"] = torch.full((3, 8, d), float("nan"), dtype=dtype, device="cuda")
    step["positions"] = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = torch.full_like(step["q"], 7.0)
    attend(step, out)
    assert step["max_query_len"] == 0 and (out == 7.0).all()
    attend({**step, "max_query_len": 2, "max_group_tokens": 4}, out)
    assert (out == 7.0).all()
    torch.cuda.synchronize()
