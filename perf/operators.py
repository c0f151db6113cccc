"""Operators for many continuations of one cached prompt, in their plain form and through the package: copies of whole cache pages (a request
is forked, a pool compacted), attention of a batch whose requests share the pages of a long prefix, and the verification of drafted
tokens against the target's probabilities.

A case names the operator (``kind``), its sizes and types; lists of lengths are texts.  ``run`` computes the plain form with elementary
operations in float32 (float64 where a border decides), or, where ``own`` is true, calls the package.  ``exact`` computes the same from the
definitions in float64, request by request: it shares the inputs with ``prepare`` and nothing else.
"""

from __future__ import annotations

import math
import struct

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _text(numbers) -> str:
    return ",".join(str(int(n)) for n in numbers)


def _numbers(text) -> list:
    return [int(part) for part in str(text).split(",") if part]


def _spread(count: int, low: int, high: int, step: int) -> str:
    """``count`` lengths between ``low`` and ``high``, uneven but fixed."""
    return _text(low + (index * step) % (high - low + 1) for index in range(count))


# --------------------------------------------------------------------------- the cases


def listed():
    return [
        # A request is forked: the page that its last tokens share with nothing yet is copied, in every layer of Qwen3-1.7B's cache.
        dict(name="pages_fork_one", kind="pages", dtype="bfloat16", runs=28, pages=96, kv_heads=8, page=16, dim=128, copies=1, sources=1),
        # Sixteen samples of one prompt: the same page to sixteen others, with heads and pages of odd sizes in the float32 path.
        dict(name="pages_fork_sixteen", kind="pages", dtype="float32", runs=5, pages=200, kv_heads=3, page=5, dim=25, copies=16, sources=1),
        # A pool is compacted: hundreds of pages move to its front.
        dict(name="pages_compact", kind="pages", dtype="bfloat16", runs=16, pages=640, kv_heads=8, page=16, dim=128, copies=256, sources=256),
        # Two samples of a short prompt, a token each: the smallest call, all latency (Qwen3-1.7B's heads).
        dict(name="prefix_two_requests", kind="attention", dtype="bfloat16", heads=16, kv_heads=8, dim=128, page=16, groups="2",
             prefix="512", queries="1,1", suffix="17,5", softcap=0.0, sink=False),
        # Thirty-two samples of one prompt in the middle of their answers (Qwen3-8B's heads).
        dict(name="prefix_samples", kind="attention", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=16, groups="32",
             prefix="4096", queries=_text([1] * 32), suffix=_spread(32, 16, 400, 61), softcap=0.0, sink=False),
        # Sixty-four requests behind one long document, the largest amount of work.
        dict(name="prefix_document", kind="attention", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=64, groups="64",
             prefix="32768", queries=_text([1] * 64), suffix=_spread(64, 1, 1024, 331), softcap=0.0, sink=False),
        # Drafted tokens being verified: portions of five and fewer tokens in three groups, one of which shares nothing, under a soft
        # cap and with a sink.
        dict(name="prefix_drafts", kind="attention", dtype="bfloat16", heads=32, kv_heads=8, dim=64, page=32, groups="8,7,1",
             prefix="2016,1024,0", queries=_text([5, 5, 4, 5, 1, 5, 5, 3] * 2), suffix=_spread(16, 9, 700, 97), softcap=30.0, sink=True),
        # The float32 path with heads of an odd size and pages that end inside every tile.
        dict(name="prefix_float32", kind="attention", dtype="float32", heads=6, kv_heads=2, dim=48, page=24, groups="5,3",
             prefix="600,264", queries="1,1,3,1,1,2,1,1", suffix="33,1,70,8,129,20,5,64", softcap=0.0, sink=False),
        # One request with three greedy drafts: the smallest verification, all latency and one read of four rows.
        dict(name="verify_one_greedy", kind="verify", vocab=151936, drafts="3", temperature="0", top_k="0", top_p="1", probabilities=False),
        # Sixteen requests without filters against a draft model's probabilities.
        dict(name="verify_draft_model", kind="verify", vocab=151936, drafts=_text([4, 4, 2, 4] * 4), temperature="0.8,1", top_k="0",
             top_p="1", probabilities=True),
        # Sixty-four requests, each with filters of its own (or none), the largest.
        dict(name="verify_filters", kind="verify", vocab=151936, drafts=_text([5, 3, 4, 1] * 16), temperature="0.7,1,0,1.3",
             top_k="50,0,0,1000", top_p="0.9,0.95,1,1", probabilities=True),
        # Drafts found by looking up the prompt (no probabilities of their own), a small vocabulary of odd size, a request without a draft.
        dict(name="verify_lookup", kind="verify", vocab=32011, drafts="7,0,2,6,1,5,3,4", temperature="1,0.6", top_k="0,40", top_p="0.9,1",
             probabilities=False),
    ]


def _log_uniform(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["pages", "attention", "attention", "verify", "verify"])
    if kind == "pages":
        copies = _log_uniform(rng, 1, 200)
        return dict(kind=kind, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), runs=rng.randint(1, 6), pages=2 * copies + rng.randint(1, 64),
                    kv_heads=rng.randint(1, 8), page=rng.choice([1, 5, 8, 16, 16, 24]), dim=rng.choice([25, 48, 64, 80, 128]), copies=copies,
                    sources=rng.choice([1, max(1, copies // 4), copies, copies]))
    if kind == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([group for group in (1, 2, 3, 4, 5, 8) if kv_heads * group <= 32])
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        dim = rng.choice([64, 128, 128, 96, 40]) if dtype == "bfloat16" else rng.choice([24, 48, 64, 128])
        page = rng.choice([1, 8, 16, 16, 24, 64, 128])
        n_groups = rng.randint(1, 3)
        groups = [_log_uniform(rng, 1, 20) for _ in range(n_groups)]
        prefix = [rng.choice([0, 1, 1, 1, 1]) * (_log_uniform(rng, 16, 8192 if dtype == "bfloat16" else 1500) // page * page) for _ in range(n_groups)]
        count = sum(groups)
        most = rng.choice([1, 1, 2, 4])
        queries = [rng.randint(1, most) for _ in range(count)]
        suffix = [n + _log_uniform(rng, 1, 500) - 1 for n in queries]
        return dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, groups=_text(groups), prefix=_text(prefix),
                    queries=_text(queries), suffix=_text(suffix), softcap=rng.choice([0.0, 0.0, 30.0]), sink=rng.choice([False, False, True]))
    count = _log_uniform(rng, 1, 40)
    filtered = rng.choice([False, True])
    return dict(kind=kind, vocab=_log_uniform(rng, 500, 151936), drafts=_text(rng.randint(0, 5) for _ in range(count)),
                temperature=rng.choice(["1", "0.7,1.2,0", "0.9,0.5"]), top_k=rng.choice(["0,20", "100", "1,0,7"]) if filtered else "0",
                top_p=rng.choice(["0.9", "0.5,1", "1,0.98,0.7"]) if filtered else "1", probabilities=rng.choice([False, True]))


# --------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEVICE)


def _starts(counts):
    total, out = 0, [0]
    for count in counts:
        total += count
        out.append(total)
    return out


def _pages_inputs(case, seed):
    """Pools of one group of layers as the cache keeps them, and the page numbers as its bookkeeping has them: on the host."""
    g = _generator(seed)
    shape = (case["runs"], case["pages"], case["kv_heads"], case["page"], case["dim"])
    dtype = DTYPES[case["dtype"]]
    keys, values = (torch.randn(shape, generator=g, device=DEVICE, dtype=dtype) for _ in range(2))
    order = torch.randperm(case["pages"], generator=g, device=DEVICE).tolist()
    copies, sources = case["copies"], case["sources"]
    destinations = order[:copies]
    first = order[copies:copies + sources]
    return dict(keys=keys, values=values, sources=[first[i * sources // copies] for i in range(copies)], destinations=destinations)


def _attention_inputs(case, seed):
    """Queries, a paged cache and the tables of a step: the pages of a group's prefix stand in every table of the group, the others
    are each request's own; pages are in no order."""
    g = _generator(seed)
    dtype, d, ps = DTYPES[case["dtype"]], case["dim"], case["page"]
    groups, prefix, queries, suffix = (_numbers(case[key]) for key in ("groups", "prefix", "queries", "suffix"))
    of_request = [index for index, count in enumerate(groups) for _ in range(count)]
    context = [prefix[of_request[r]] + suffix[r] for r in range(len(queries))]
    shared = [length // ps for length in prefix]
    needed = [(length + ps - 1) // ps for length in context]
    total = sum(shared) + sum(n - shared[of_request[r]] for r, n in enumerate(needed)) + 3
    order = torch.randperm(total, generator=g, device=DEVICE).tolist()
    width, at, tables = max(needed), 0, []
    group_pages = []
    for count in shared:
        group_pages.append(order[at:at + count])
        at += count
    for r, n in enumerate(needed):
        pages = group_pages[of_request[r]]
        own_pages = order[at:at + n - len(pages)]
        at += len(own_pages)
        tables.append(pages + own_pages + [total - 1] * (width - n))
    query_start = _starts(queries)
    positions = [context[r] - queries[r] + i for r in range(len(queries)) for i in range(queries[r])]
    group_start = _starts(groups)
    pool = (total, case["kv_heads"], ps, d)
    tokens = [query_start[b] - query_start[a] for a, b in zip(group_start[:-1], group_start[1:])]
    return dict(
        q=(1.5 * torch.randn(query_start[-1], case["heads"], d, generator=g, device=DEVICE)).to(dtype),
        k_pool=torch.randn(pool, generator=g, device=DEVICE, dtype=dtype), v_pool=torch.randn(pool, generator=g, device=DEVICE, dtype=dtype),
        sink=torch.randn(case["heads"], generator=g, device=DEVICE) if case["sink"] else None,
        block_tables=_ints(sum(tables, [])).view(len(tables), width), positions=_ints(positions), query_start=_ints(query_start),
        context_lens=_ints(context), group_start=_ints(group_start), prefix_lens=_ints(prefix), scale=d ** -0.5,
        softcap=case["softcap"] or None,
        # upper bounds that the host knows: tokens of a request and of a group, keys of a prefix and behind it
        bounds=dict(max_query_len=max(queries), max_group_tokens=max(tokens), max_prefix_len=max(prefix), max_suffix_len=max(suffix)))


def _cycled(text, count, kind):
    parts = str(text).split(",")
    return [kind(parts[index % len(parts)]) for index in range(count)]


def _verify_inputs(case, seed):
    """Logits of a target whose mass lies on some hundred tokens, drafts drawn from a nearby distribution, the random numbers, and the sampling
    records of the requests' slots (temperature, top-p, top-k as ``kernels.sample`` takes them)."""
    g = _generator(seed)
    drafts, vocab = _numbers(case["drafts"]), case["vocab"]
    count, total = len(drafts), sum(drafts)
    temperature, top_p, top_k = _cycled(case["temperature"], count, float), _cycled(case["top_p"], count, float), _cycled(case["top_k"], count, int)
    logits = 2.0 * torch.randn(total + count, vocab, generator=g, device=DEVICE)
    head = torch.randint(vocab, (total + count, 12), generator=g, device=DEVICE)
    logits.scatter_reduce_(1, head, 14.0 - 4.0 * torch.rand(total + count, 12, generator=g, device=DEVICE), "amax")
    starts = _starts(drafts)
    rows = [starts[r] + r + i for r in range(count) for i in range(drafts[r])]
    near = logits[rows] + 0.7 * torch.randn(total, vocab, generator=g, device=DEVICE)
    probs = torch.exp(near - near.amax(-1, keepdim=True) if total else near)
    probs = probs / probs.sum(-1, keepdim=True)
    chosen = (probs / torch.empty_like(probs).exponential_(generator=g)).argmax(-1).int() if total else _ints([])
    if not case["probabilities"]:
        # a lookup proposes what the target finds likely now and then
        likely = logits[rows].argmax(-1).int() if total else chosen
        chosen = torch.where(torch.rand(total, generator=g, device=DEVICE) < 0.6, likely, chosen)
    slots = torch.randperm(count + 1, generator=g, device=DEVICE)[:count].tolist()
    records = [[0] * 8 for _ in range(count + 1)]
    for r, slot in enumerate(slots):
        records[slot] = list(struct.unpack("<8i", struct.pack("<ffiIIiii", temperature[r], top_p[r], top_k[r], 1, 0, 0, 0, 0)))
    as_float = lambda values: torch.tensor(values, dtype=torch.float32, device=DEVICE)
    return dict(
        logits=logits, drafts=chosen, draft_start=_ints(starts), draft_probs=probs if case["probabilities"] else None,
        uniforms=torch.rand(total, generator=g, device=DEVICE), noise=torch.empty(count, vocab, device=DEVICE).exponential_(generator=g),
        records=_ints(sum(records, [])).view(count + 1, 8), slots=_ints(slots), temperature=as_float(temperature), top_p=as_float(top_p),
        top_k=_ints(top_k), most=max(drafts), filtered=any(k > 0 for k in top_k) or any(p < 1.0 for p in top_p),
        accepted=_ints([0] * count), next_token=_ints([0] * count), target_probs=torch.zeros(total, device=DEVICE))


INPUTS = {"pages": _pages_inputs, "attention": _attention_inputs, "verify": _verify_inputs}


def prepare(case, seed):
    return dict(INPUTS[case["kind"]](case, seed), kind=case["kind"])


# --------------------------------------------------------------------------- one pass


def run(state):
    return {"pages": _run_pages, "attention": _run_attention, "verify": _run_verify}[state["kind"]](state)


def _run_pages(s):
    keys, values = s["keys"], s["values"]
    if own:
        from miniserve_b200 import kernels

        kernels.copy_pages([keys, values], s["sources"], s["destinations"])
    else:
        sources = torch.tensor(s["sources"], device=keys.device)
        destinations = torch.tensor(s["destinations"], device=keys.device)
        keys[:, destinations] = keys[:, sources]
        values[:, destinations] = values[:, sources]
    return {"keys": keys, "values": values}


def _run_attention(s):
    if own:
        from miniserve_b200 import kernels

        out = torch.empty_like(s["q"])
        kernels.shared_prefix_attention(s["q"], s["k_pool"], s["v_pool"], s["block_tables"], s["positions"], s["query_start"],
                                        s["context_lens"], s["group_start"], s["prefix_lens"], scale=s["scale"], out=out,
                                        softcap=s["softcap"], sink=False if s["sink"] is None else s["sink"], **s["bounds"])
        return {"out": out}
    starts = s["query_start"].long()
    group_start = s["group_start"].long()
    bounds, tables = s["bounds"], s["block_tables"].long()
    prefix, context = s["prefix_lens"].long(), s["context_lens"].long()
    n_requests = context.numel()
    group_of_request = torch.searchsorted(group_start, torch.arange(n_requests, device=starts.device), right=True) - 1
    # the prefix: the tokens of a group's requests against the pages that its first request names
    first_token = starts[group_start]
    seen = _part(s, first_token, bounds["max_group_tokens"], tables[group_start[:-1]], torch.zeros_like(prefix), prefix, bounds["max_prefix_len"])
    # what lies behind it, request by request
    behind = _part(s, starts, bounds["max_query_len"], tables, prefix[group_of_request], context, bounds["max_suffix_len"])
    top = torch.maximum(seen[0], behind[0])
    if s["sink"] is not None:
        top = torch.maximum(top, s["sink"])
    shift = lambda part: torch.exp(part[0] - top)
    total = shift(seen) * seen[1] + shift(behind) * behind[1]
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"] - top)
    out = (shift(seen)[..., None] * seen[2] + shift(behind)[..., None] * behind[2]) / total[..., None]
    return {"out": out.to(s["q"].dtype)}


def _part(s, starts, most_tokens, tables, first_key, last_key, most_keys):
    """Attention of blocks of consecutive tokens (``starts``: their borders) to the keys first_key .. last_key - 1 that each block's table names: per
    token and head the largest score, the sum of the exponentials relative to it and the sum of the values weighted with them."""
    q, ps = s["q"].float(), s["k_pool"].shape[2]
    n, n_q, d = q.shape
    n_kv, device = s["k_pool"].shape[1], q.device
    blocks = starts.numel() - 1
    token = starts[:-1, None] + torch.arange(most_tokens, device=device)
    token = torch.minimum(token, (starts[1:, None] - 1).clamp(min=0))
    key = first_key[:, None] + torch.arange(most_keys, device=device)
    page = torch.gather(tables, 1, (key // ps).clamp(max=tables.shape[1] - 1))
    keys = s["k_pool"][page, :, key % ps].float().transpose(1, 2)                           # [blocks, n_kv, keys, d]
    values = s["v_pool"][page, :, key % ps].float().transpose(1, 2)
    mine = q[token].view(blocks, most_tokens, n_kv, n_q // n_kv, d).permute(0, 2, 1, 3, 4).reshape(blocks, n_kv, most_tokens * (n_q // n_kv), d)
    scores = torch.matmul(mine, keys.transpose(2, 3)).view(blocks, n_kv, most_tokens, n_q // n_kv, most_keys) * s["scale"]
    if s["softcap"]:
        scores = s["softcap"] * torch.tanh(scores / s["softcap"])
    visible = (key[:, None, :] < last_key[:, None, None]) & (key[:, None, :] <= s["positions"].long()[token][:, :, None])
    scores = scores.masked_fill(~visible[:, None, :, None, :], -math.inf)
    if most_keys:
        top = scores.amax(-1)
        weights = torch.exp(scores - torch.where(top > -math.inf, top, 0.0)[..., None])
    else:
        top, weights = torch.full(scores.shape[:-1], -math.inf, device=device), scores
    sums = weights.sum(-1)
    mixed = torch.matmul(weights.reshape(blocks, n_kv, most_tokens * (n_q // n_kv), most_keys), values).view(blocks, n_kv, most_tokens, n_q // n_kv, d)
    # back to the order of the tokens
    at = torch.arange(n, device=device)
    block = torch.searchsorted(starts, at, right=True) - 1
    pick = lambda x: x.transpose(1, 2)[block, at - starts[block]].reshape((n, n_q) + tuple(x.shape[4:]))
    return pick(top), pick(sums), pick(mixed)


def _run_verify(s):
    if own:
        from miniserve_b200 import kernels

        kernels.verify_drafts(s["logits"], s["drafts"], s["draft_start"], s["uniforms"], s["noise"], s["accepted"], s["next_token"],
                              draft_probs=s["draft_probs"], records=s["records"], slot_of_request=s["slots"], target_probs=s["target_probs"])
        return {"accepted": s["accepted"], "next_token": s["next_token"], "target_probs": s["target_probs"]}
    logits, starts, drafts = s["logits"], s["draft_start"].long(), s["drafts"].long()
    rows, vocab = logits.shape
    device = logits.device
    count, total = starts.numel() - 1, drafts.numel()
    row_start = starts + torch.arange(count + 1, device=device)
    request = torch.searchsorted(row_start, torch.arange(rows, device=device), right=True) - 1
    greedy = s["temperature"][request] == 0.0
    heat = torch.where(greedy, 1.0, s["temperature"][request])[:, None]
    if s["filtered"]:
        # (where a token's membership hangs on a sum's last bits, in float64)
        x = logits.double()
        weights = torch.exp((x - x.amax(-1, keepdim=True)) / heat.double())
        ranked, order = torch.sort(x, dim=-1, descending=True, stable=True)
        top_k = torch.where(s["top_k"] > 0, s["top_k"], vocab).long()[request][:, None]
        kept = torch.arange(vocab, device=device)[None, :] < top_k
        mass = torch.gather(weights, 1, order) * kept
        before = torch.cumsum(mass, -1) - mass
        limit = s["top_p"].double()[request][:, None]
        kept = kept & ((before <= limit * mass.sum(-1, keepdim=True)) | (limit >= 1.0))
        keep = torch.zeros_like(kept).scatter_(1, order, kept)
        weights = (weights * keep).float()
    else:
        weights = torch.exp((logits - logits.amax(-1, keepdim=True)) / heat)
    probs = weights / weights.sum(-1, keepdim=True)
    best = torch.zeros_like(probs).scatter_(1, logits.argmax(-1, keepdim=True), 1.0)
    probs = torch.where(greedy[:, None], best, probs)
    # which drafts pass: u q < p, and all before them
    owner = torch.searchsorted(starts, torch.arange(total, device=device), right=True) - 1
    draft_row = torch.arange(total, device=device) + owner
    target = probs[draft_row, drafts]
    theirs = s["draft_probs"][torch.arange(total, device=device), drafts] if s["draft_probs"] is not None else torch.ones_like(target)
    passes = torch.where(greedy[draft_row], target > 0.0, s["uniforms"] * theirs < target)
    table = torch.zeros((count, s["most"] + 1), dtype=torch.bool, device=device)
    table[owner, torch.arange(total, device=device) - starts[owner]] = passes
    accepted = torch.cumprod(table.long(), -1).sum(-1)
    # the row that decides the next token, and what the draft leaves of it
    row = row_start[:-1] + accepted
    rejected = accepted < starts[1:] - starts[:-1]
    left = probs[row]
    if total:
        draft = (starts[:-1] + accepted).clamp(max=total - 1)
        if s["draft_probs"] is not None:
            less = (left - s["draft_probs"][draft]).clamp(min=0.0)
        else:
            less = left.scatter(1, drafts[draft][:, None], 0.0)
        usable = (rejected & ~greedy[row] & (less > 0.0).any(-1))[:, None]
        left = torch.where(usable, less, left)
    next_token = torch.where(greedy[row], left.argmax(-1), (left / s["noise"]).argmax(-1))
    return {"accepted": accepted.int(), "next_token": next_token.int(), "target_probs": target}


# --------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["kind"] == "pages":
        page = case["kv_heads"] * case["page"] * case["dim"] * (2 if case["dtype"] == "bfloat16" else 4)
        return {"bytes": 2 * case["runs"] * page * (case["sources"] + case["copies"]), "flops": 0}
    if case["kind"] == "attention":
        size = 2 if case["dtype"] == "bfloat16" else 4
        groups, prefix, queries, suffix = (_numbers(case[key]) for key in ("groups", "prefix", "queries", "suffix"))
        of_request = [index for index, count in enumerate(groups) for _ in range(count)]
        keys = sum(prefix) + sum(suffix)
        pairs = sum(sum(prefix[of_request[r]] + suffix[r] - i for i in range(queries[r])) for r in range(len(queries)))
        return {"bytes": size * (2 * sum(queries) * case["heads"] * case["dim"] + 2 * keys * case["kv_heads"] * case["dim"]),
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    drafts = _numbers(case["drafts"])
    rows, count = sum(drafts) + len(drafts), len(drafts)
    temperature = _cycled(case["temperature"], count, float)
    noisy = sum(t > 0.0 for t in temperature)
    compared = sum(t > 0.0 and n > 0 for t, n in zip(temperature, drafts)) if case["probabilities"] else 0
    return {"bytes": 4 * case["vocab"] * (rows + noisy + compared), "flops": 4 * case["vocab"] * (rows + 2 * noisy)}


# --------------------------------------------------------------------------- the same from the definitions, in float64


def exact(case, seed):
    inputs = INPUTS[case["kind"]](case, seed)
    return {"pages": _exact_pages, "attention": _exact_attention, "verify": _exact_verify}[case["kind"]](inputs)


def _exact_pages(s):
    out = {}
    for name in ("keys", "values"):
        pool = s[name].clone()
        for source, destination in zip(s["sources"], s["destinations"]):
            pool[:, destination] = s[name][:, source]
        out[name] = pool
    return out


def _exact_attention(s):
    tables, starts, context = s["block_tables"].tolist(), s["query_start"].tolist(), s["context_lens"].tolist()
    ps = s["k_pool"].shape[2]
    n, n_q, d = s["q"].shape
    group = n_q // s["k_pool"].shape[1]
    out = torch.empty(n, n_q, d, dtype=torch.float64, device=s["q"].device)
    for r, length in enumerate(context):
        pages = torch.tensor(tables[r][:(length + ps - 1) // ps], device=s["q"].device)
        keys, values = (pool[pages].transpose(1, 2).reshape(-1, pool.shape[1], d)[:length].double().repeat_interleave(group, 1)
                        for pool in (s["k_pool"], s["v_pool"]))
        for token in range(starts[r], starts[r + 1]):
            last = length - (starts[r + 1] - token) + 1
            scores = torch.einsum("hd,khd->hk", s["q"][token].double(), keys[:last]) * s["scale"]
            if s["softcap"]:
                scores = s["softcap"] * torch.tanh(scores / s["softcap"])
            if s["sink"] is not None:
                scores = torch.cat([scores, s["sink"].double()[:, None]], 1)
            share = torch.softmax(scores, -1)[:, :last]
            out[token] = torch.einsum("hk,khd->hd", share, values[:last])
    return {"out": out}


def _exact_verify(s):
    starts, drafts = s["draft_start"].tolist(), s["drafts"].tolist()
    temperature, top_k = s["temperature"].tolist(), s["top_k"].tolist()
    top_p = s["top_p"].double().tolist()
    vocab = s["logits"].shape[1]

    def distribution(row, r):
        x = s["logits"][row].double()
        if temperature[r] == 0.0:
            p = torch.zeros_like(x)
            p[int(s["logits"][row].argmax())] = 1.0
            return p
        p = torch.softmax(x / temperature[r], -1)
        order = torch.sort(x, descending=True, stable=True).indices
        if 0 < top_k[r] < vocab:
            p[order[top_k[r]:]] = 0.0
            p = p / p.sum()
        if top_p[r] < 1.0:
            sorted_p = p[order]
            p[order[sorted_p.cumsum(-1) - sorted_p > top_p[r]]] = 0.0
            p = p / p.sum()
        return p

    accepted, next_token, target = [], [], []
    for r in range(len(starts) - 1):
        row, taken, draw_from = starts[r] + r, 0, None
        for i in range(starts[r], starts[r + 1]):
            p = distribution(row + i - starts[r], r)
            target.append(float(p[drafts[i]]))
            if draw_from is not None:
                continue
            q = s["draft_probs"][i].double() if s["draft_probs"] is not None else torch.zeros_like(p).index_fill_(0, s["drafts"][i:i + 1].long(), 1.0)
            passes = target[-1] > 0.0 if temperature[r] == 0.0 else float(s["uniforms"][i]) * float(q[drafts[i]]) < target[-1]
            if passes:
                taken += 1
            elif temperature[r] == 0.0:
                draw_from = p
            else:
                less = (p - q).clamp(min=0.0)
                draw_from = less if bool((less > 0.0).any()) else p
        if draw_from is None:
            draw_from = distribution(row + taken, r)
        accepted.append(taken)
        next_token.append(int((draw_from if temperature[r] == 0.0 else draw_from / s["noise"][r].double()).argmax()))
    return {"accepted": _ints(accepted), "next_token": _ints(next_token), "target_probs": torch.tensor(target, dtype=torch.float64, device=DEVICE)}
