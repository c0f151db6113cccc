"""The step function: one batch of (request, its next tokens) through the model, from the cache.

A step's entries may be portions of prompts of any length beside single decoded tokens.  They
are flattened into one batch (no padding), every index a kernel will use is checked on the
host (miniserve/engine/flat_batch.py:490-569 does the same for its decode rows), the index
arrays travel to the device in one copy, the model runs once over all tokens, and the logits
come back only for the positions that were asked for.  MiniServe runs a step as one forward
per prompt portion plus one for the decode rows (miniserve/engine/executor.py:239-255) and
computes logits for every position of a portion; this engine does neither.
"""

from __future__ import annotations

from dataclasses import dataclass, field
from typing import Optional, Sequence

import torch

from .. import kernels
from ..cache.manager import RELEASED, CacheManager, StepReservation
from ..parts.base import PagedKVNeed
from ..parts.context import SharedPrefixes, StepContext


@dataclass
class StepEntry:
    """A request's next tokens and the indices among them whose logits are wanted."""

    request_id: str
    tokens: Sequence[int]
    want: Sequence[int] = field(default_factory=tuple)


DECODE_BUCKETS = (1, 2, 4, 8, 16, 32, 64, 128, 256)

# With ``shared_prefixes``: keys of a prefix from which on requests form a group, and keys that need not be read a second time from which on a step
# goes that way - one that runs eagerly anyway, and one that a captured graph would run, whose launches cost the host nothing.  Qwen3-1.7B, bfloat16, ms
# a step, without / with: four tokens each of 2 requests behind 512 keys 2.9 / 2.7, of 63 5.2 / 5.3, of 32 behind 8,192 6.2 / 5.0, of 63 behind 16,000
# 18.4 / 6.8; a token each, replayed / eager and shared: 32 behind 2,048 2.7 / 4.6, 63 behind 2,048 3.7 / 5.3, 8 behind 16,000 3.5 / 3.1, 32 behind 8,192
# 5.7 / 5.0, 63 behind 8,192 9.8 / 5.9, 63 behind 16,000 17.6 / 6.8.
SHARED_KEYS_LEAST, SHARED_KEYS_EAGER, SHARED_KEYS_REPLAYED = 128, 512, 200_000

# What else those keys have to outweigh, in keys: tokens of requests that bring several, whose own keys go through kernels made for few rows and whose results
# through float32 parts (SHARED_KEYS_TOKEN for each, SHARED_KEYS_PAIR for each pair of a request's, both for each query head of a key head), and, where a request brings more than 16
# rows to a key head, the longest way along one request's own keys, which are then not cut into parts (SHARED_KEYS_OWN for each, with eight key heads; fewer
# read less for every key).  us of one layer's attention, without / with sharing, 16 query and 8 key heads of 128, bfloat16: eight requests behind 2,048 keys, 1
# token each 14 / 11, 16 each 22 / 19, 64 each 23 / 39, 512 each 92 / 262; behind 8,192, 64 each 66 / 57, 256 each 132 / 203; 63 single tokens behind 2,048
# beside another request's portion of 64 89 / 21, of 512 92 / 77, of 2,048 109 / 354; behind 8,192 beside 2,048 324 / 377.  Over 2,064 steps of six sets of
# heads, behind 512 to 16,384 keys, the steps chosen gain 74 of the 85 ms that the faster way of each would, 37 are behind by
# more than 5 % (0.4 ms in all, 1.57 times as long at worst); every step from SHARED_KEYS_EAGER on would have lost 174.
SHARED_KEYS_TOKEN, SHARED_KEYS_PAIR, SHARED_KEYS_OWN = 60, 0.05, 160


def prefix_groups(common: Sequence[int], least: int) -> tuple[int, list[tuple[int, int]]]:
    """Requests in their order, cut into groups of neighbours so that the most keys need not be read a second time: ``(that number, [(requests, shared
    keys)])``.  ``common[i]``: keys that request i has in common with the one before it; a group shares the fewest of those between its
    requests, a group of one and one that would share fewer than ``least`` nothing.

    The best cut of the first requests is the best of an earlier place and one more group.  Of neighbours that all have the same number in common, a cut
    goes to the first or the last pair (what one group wins as it moves along, the other loses), so that places between need no look."""
    n = len(common)
    places = [0] + [i for i in range(1, n) if i == 1 or i == n - 1 or not common[i - 1] == common[i] == common[i + 1]] + [n]
    saved, before, shared = [0], [0], [0]
    for at in range(1, len(places)):
        end, fewest = places[at], None                    # fewest: between the requests of the group from places[start] to end
        most = -1
        for start in range(at - 1, -1, -1):
            first = places[start]
            if start + 1 < at:
                fewest = common[places[start + 1]] if fewest is None else min(fewest, common[places[start + 1]])
            elif end - first > 1:
                fewest = common[first + 1]
            keys = fewest if fewest is not None and fewest >= least else 0
            value = saved[start] + (end - first - 1) * keys
            if value > most:
                most, source, kept = value, start, keys
            if fewest is not None and (fewest < least or saved[start] + (end - 1) * fewest <= most):
                break                                     # (no earlier start can be better)
        saved.append(most), before.append(source), shared.append(kept)
    groups, at = [], len(places) - 1
    while at > 0:
        count = places[at] - places[before[at]]
        groups += [(count, shared[at])] if shared[at] else [(1, 0)] * count
        at = before[at]
    return saved[-1], groups[::-1]


class DecodeGraph:
    """One captured decode step for exactly ``rows`` rows, with fixed device buffers.

    Mechanics of miniserve/engine/graph.py:645-823: the index arrays live in one static buffer
    that a replay overwrites with a single copy; rows beyond the live ones are padding that reads
    and writes only the pool's scratch page; positions feed the rotation inside the graph, so
    nothing about a position is baked in; the pools never move.  Unlike there, every batch size
    up to the largest bucket replays a graph (the next bucket up, padded).
    """

    def __init__(self, step_function: "StepFunction", rows: int) -> None:
        sf = step_function
        self.rows = rows
        manager, storage = sf.manager, sf.storage
        ps = self.page_size = manager.page_size
        self.width = (sf.max_model_len + ps - 1) // ps
        n_groups = len(manager.paged_needs)
        # layout: tokens, positions, request_of_token, query_start, context_lens, state_slots, logit_rows,
        #         draw_index, then per group (block_tables, slots)
        sizes = [rows, rows, rows, rows + 1, rows, rows, rows, rows] + [rows * self.width, rows] * n_groups
        self.offsets = [0]
        for size in sizes:
            self.offsets.append(self.offsets[-1] + size)
        self.host = torch.empty(self.offsets[-1], dtype=torch.int32, pin_memory=True)
        self.host_np = self.host.numpy()             # same memory, cheaper to fill from Python lists
        self.live_rows = -1
        self.copied: Optional[torch.cuda.Event] = None     # recorded after the last copy of the host mirror
        # per row: (the request's cache record, pages of its committed table that the mirror shows, per group, pages given back, per
        # group, and the record's count of changes to committed pages)
        self.row_owner: list = [None] * rows
        # groups whose pages can be given back behind a window or a chunk: a row's table may change anywhere between two steps
        self.gives_back = [not need.keeps_all for need in manager.paged_needs]
        self.meta = torch.zeros(self.offsets[-1], dtype=torch.int32, device=sf.device)
        self.n_groups = n_groups
        self.scratch = storage.scratch_page
        self.scratch_slot = storage.scratch_slot
        self._fill_padding(0)
        self.meta.copy_(self.host)
        views = [self.meta[self.offsets[i]:self.offsets[i + 1]] for i in range(len(sizes))]
        group_views = [(views[8 + 2 * g].view(rows, self.width), views[9 + 2 * g]) for g in range(n_groups)]
        self.ctx_args = dict(
            n_tokens=rows, n_requests=rows, token_ids=views[0], positions=views[1], request_of_token=views[2],
            query_start=views[3], context_lens=views[4], state_slots=views[5], logit_rows=views[6],
            max_query_len=1, max_context_len=sf.max_model_len, dtype=sf.model.dtype, device=sf.device,
            group_views=group_views)
        self.draw_index = views[7]
        self.tokens_out = torch.zeros(rows, dtype=torch.int32, device=sf.device)
        self.logits: Optional[torch.Tensor] = None
        self.graph = torch.cuda.CUDAGraph()
        self.kernel_launches = 0

        def body() -> torch.Tensor:
            ctx = StepContext(**self.ctx_args)
            logits = sf.model.forward(ctx, storage)
            kernels.sample(logits, storage.sampling_records, ctx.state_slots, self.draw_index, self.tokens_out)
            return logits

        side = torch.cuda.Stream(device=sf.device)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            body()                       # warm-up outside the capture (lazy library set-up happens here)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        before = kernels.launch_count
        with torch.cuda.graph(self.graph, pool=sf.graph_pool):
            self.logits = body()
        self.kernel_launches = kernels.launch_count - before

    def _fill_padding(self, first_row: int) -> None:
        """Rows from ``first_row`` on become padding: token 0 at position 0 on the scratch page, in the scratch slot."""
        import numpy

        o, rows, host = self.offsets, self.rows, self.host_np
        ps = self.page_size
        host[o[0] + first_row:o[1]] = 0
        host[o[1] + first_row:o[2]] = 0
        host[o[2]:o[3]] = numpy.arange(rows, dtype=numpy.int32)
        host[o[3]:o[4]] = numpy.arange(rows + 1, dtype=numpy.int32)
        host[o[4] + first_row:o[5]] = 1
        host[o[5] + first_row:o[6]] = self.scratch_slot
        host[o[6]:o[7]] = numpy.arange(rows, dtype=numpy.int32)
        host[o[7] + first_row:o[8]] = 0
        for g in range(self.n_groups):
            tables = host[o[8 + 2 * g]:o[9 + 2 * g]].reshape(rows, self.width)
            tables[first_row:] = self.scratch
            host[o[9 + 2 * g] + first_row:o[10 + 2 * g]] = self.scratch * ps


class StepFunction:
    def __init__(self, model, storage, manager: CacheManager, max_model_len: int, use_graphs: bool = False,
                 shared_prefixes: bool = False) -> None:
        self.model, self.storage, self.manager = model, storage, manager
        # the paged groups whose steps may read shared prefixes once
        self.sharing_groups: dict[int, int] = {} if not shared_prefixes else {
            manager.group_index[group][1]: heads for group, heads in model.sharing_groups().items() if manager.group_index[group][0] == "paged"}
        self.max_model_len = max_model_len
        self.device = model.device
        self.vocab_size = model.spec.vocab_size
        self.use_graphs = use_graphs
        self.graphs: dict[int, DecodeGraph] = {}
        self.graph_pool = None
        self.graph_replays = 0
        self.eager_steps = 0
        self.last_tokens: Optional[torch.Tensor] = None   # tokens sampled inside the last replayed graph
        self.last_graph: Optional[DecodeGraph] = None

    # ------------------------------------------------------------------ batch building
    def build_context(self, entries: Sequence[StepEntry], reservation: StepReservation) -> StepContext:
        import numpy

        manager, ps = self.manager, self.manager.page_size
        if len(entries) != len(reservation.items):
            raise ValueError("the reservation was made for other entries")
        int32 = numpy.int32
        token_parts, position_parts, request_parts, slot_parts = [], [], [], None
        query_start = [0]
        context_lens: list[int] = []
        state_slots: list[int] = []
        logit_rows: list[int] = []
        n_groups = len(manager.paged_needs)
        slot_parts = [[] for _ in range(n_groups)]
        width = 1
        n = 0
        for row, (entry, item) in enumerate(zip(entries, reservation.items)):
            count = len(entry.tokens)
            if entry.request_id != item.request_id or count != item.end - item.start:
                raise ValueError(f"entry {row} does not match its reservation")
            if item.end > self.max_model_len:
                raise ValueError(f"request {entry.request_id!r} would reach {item.end} tokens; the limit is {self.max_model_len}")
            ids = numpy.asarray(entry.tokens, dtype=numpy.int64)      # (no copy if the caller holds its tokens as such an array)
            if count and (int(ids.min()) < 0 or int(ids.max()) >= self.vocab_size):
                raise ValueError(f"a token id of request {entry.request_id!r} lies outside the vocabulary of {self.vocab_size}")
            for index in entry.want:
                if not 0 <= index < count:
                    raise ValueError(f"wanted index {index} outside the {count} tokens of the entry")
                logit_rows.append(n + index)
            token_parts.append(ids.astype(int32))
            position_parts.append(numpy.arange(item.start, item.end, dtype=int32))
            request_parts.append(numpy.full(count, row, dtype=int32))
            n += count
            query_start.append(n)
            context_lens.append(item.end)
            state_slots.append(manager.requests[entry.request_id].slot)
            for group in range(n_groups):
                slot_parts[group].append(numpy.asarray(item.slots[group], dtype=int32))
                width = max(width, len(item.tables[group]))

        scratch = self.storage.scratch_page
        limit = self.storage.num_pages
        r = len(entries)
        tables = []
        slots = []
        for group in range(n_groups):
            table = numpy.full((r, width), scratch, dtype=int32)
            for row, item in enumerate(reservation.items):
                pages = numpy.asarray(item.tables[group], dtype=int32)
                pages = numpy.where(pages == RELEASED, scratch, pages)
                if pages.size and (int(pages.min()) < 0 or int(pages.max()) > limit):
                    raise ValueError(f"a page of request {item.request_id!r} lies outside the pool of {limit}")
                table[row, :pages.size] = pages
            tables.append(table.reshape(-1))
            group_slots = numpy.concatenate(slot_parts[group]) if slot_parts[group] else numpy.zeros(0, dtype=int32)
            if group_slots.size and (int(group_slots.min()) < 0 or int(group_slots.max()) >= limit * ps):
                raise ValueError("a slot lies outside the pool")
            slots.append(group_slots)

        empty = numpy.zeros(0, dtype=int32)
        pieces = [numpy.concatenate(token_parts) if token_parts else empty,
                  numpy.concatenate(position_parts) if position_parts else empty,
                  numpy.concatenate(request_parts) if request_parts else empty,
                  numpy.asarray(query_start, dtype=int32), numpy.asarray(context_lens, dtype=int32),
                  numpy.asarray(state_slots, dtype=int32), numpy.asarray(logit_rows, dtype=int32)]
        for group in range(n_groups):
            pieces += [tables[group], slots[group]]
        total = sum(p.size for p in pieces)
        staging = torch.empty(max(total, 1), dtype=torch.int32, pin_memory=self.device.type == "cuda")
        staging_np = staging.numpy()
        offset = 0
        spans = []
        for piece in pieces:
            staging_np[offset:offset + piece.size] = piece
            spans.append((offset, piece.size))
            offset += piece.size
        on_device = staging.to(self.device, non_blocking=True)
        views = [on_device[start:start + length] for start, length in spans]
        group_views = []
        for group in range(n_groups):
            group_views.append((views[7 + 2 * group].view(r, width), views[8 + 2 * group]))
        shared_prefixes = []
        if self.sharing_groups:
            ids = [e.request_id for e in entries]
            sharing = [self._shared_groups(ids, group, SHARED_KEYS_EAGER) if group in self.sharing_groups else None for group in range(n_groups)]
            sharing = [found if found is not None and self._outweighs(found, group, query_start, context_lens) else None for group, found in enumerate(sharing)]
            if any(found is not None for found in sharing):
                shared_prefixes = [None if found is None else self._share(found, query_start, context_lens) for found in sharing]
        return StepContext(
            shared_prefixes=shared_prefixes, n_tokens=n, n_requests=r, token_ids=views[0], positions=views[1], request_of_token=views[2],
            query_start=views[3], context_lens=views[4], state_slots=views[5], logit_rows=views[6],
            max_query_len=max((len(e.tokens) for e in entries), default=0),
            max_context_len=max(context_lens, default=0), dtype=self.model.dtype, device=self.device,
            host_query_start=query_start, host_context_lens=context_lens, host_state_slots=state_slots,
            group_views=group_views)

    # ------------------------------------------------------------------ forks and moves of what the cache holds
    def fork(self, request_id: str, new_ids: Sequence[str]) -> None:
        """Continuations of a request as it stands (samples of one prompt, drafts to compare): ``new_ids`` share its full pages and get a copy
        of the page that is partly filled.  Their sampling records are the caller's to write (``storage.reset_slot``)."""
        new_ids = list(new_ids)
        copies = self.manager.fork(request_id, new_ids)
        try:
            self.storage.copy_pages(copies)
        except BaseException:
            for new_id in new_ids:
                self.manager.release(new_id)
            raise

    def compact(self) -> None:
        """Moves the pages in use to the front of their pools."""
        copies = self.manager.compact()
        try:
            self.storage.copy_pages(copies)
        except BaseException:
            self.manager.take_back(copies)
            raise

    # ------------------------------------------------------------------ prefixes that a step's requests share
    def _shared_groups(self, ids: Sequence[str], group: int, least: int) -> Optional[list[tuple[int, int]]]:
        """(requests, shared keys) of the groups that a step's requests form in one paged group, in their order; None where fewer than ``least`` keys
        need not be read a second time, or a window or another form of cache does not allow it."""
        manager = self.manager
        if not isinstance(manager.paged_needs[group], PagedKVNeed) or not manager.paged_needs[group].keeps_all:
            return None
        common = [manager.shared_pages(ids[i - 1], ids[i])[group] * manager.page_size if i else 0 for i in range(len(ids))]
        saved, groups = prefix_groups(common, SHARED_KEYS_LEAST)
        return groups if saved >= least else None

    def _outweighs(self, groups: Sequence[tuple[int, int]], group: int, query_start: Sequence[int], context_lens: Sequence[int]) -> bool:
        """Whether the keys that need not be read a second time outweigh what else is slower (see SHARED_KEYS_TOKEN)."""
        heads = self.sharing_groups[group]
        new = [end - start for start, end in zip(query_start[:-1], query_start[1:])]
        most = heads * sum(SHARED_KEYS_TOKEN * count + SHARED_KEYS_PAIR * count * count for count in new if count > 1)
        if max(new) * heads > 16:
            prefix = [keys for count, keys in groups for _ in range(count)]
            most += SHARED_KEYS_OWN * 8 / self.manager.paged_needs[group].num_kv_heads * max(length - keys for length, keys in zip(context_lens, prefix))
        return sum((count - 1) * keys for count, keys in groups) >= most

    def _share(self, groups: Sequence[tuple[int, int]], query_start: Sequence[int], context_lens: Sequence[int]) -> SharedPrefixes:
        starts, tokens, behind = [0], 0, 0
        for count, keys in groups:
            first = starts[-1]
            starts.append(first + count)
            tokens = max(tokens, query_start[first + count] - query_start[first])
            behind = max(behind, max(context_lens[first:first + count]) - keys)
        staging = torch.tensor(starts + [keys for _, keys in groups], dtype=torch.int32, pin_memory=self.device.type == "cuda")
        on_device = staging.to(self.device, non_blocking=True)
        return SharedPrefixes(on_device[:len(starts)], on_device[len(starts):], tokens, max(keys for _, keys in groups), behind)

    # ------------------------------------------------------------------ running
    def replays(self, entries: Sequence[StepEntry]) -> bool:
        """Whether these entries run as a captured graph: single tokens, all of whose logits are wanted, that share no prefix long enough to be worth
        an eager step."""
        single = bool(self.use_graphs and entries and len(entries) <= DECODE_BUCKETS[-1]
                      and all(len(e.tokens) == 1 and list(e.want) == [0] for e in entries))
        if single and self.sharing_groups and len(entries) > 1:
            ids = [e.request_id for e in entries]
            return all(self._shared_groups(ids, group, SHARED_KEYS_REPLAYED) is None for group in self.sharing_groups)
        return single

    def run(self, entries: Sequence[StepEntry], reservation: StepReservation,
            draw_index: Optional[Sequence[int]] = None, feed_back: bool = False) -> torch.Tensor:
        """float32 logits ``[number of wanted positions, vocab]`` on the device, in entry order.

        A step of single tokens whose logits are all wanted replays a captured graph when graphs
        are on; the graph also samples, and ``last_tokens`` then holds one token per entry
        (``draw_index``: each request's draw count, for its random stream).  ``feed_back``: the
        entries are the rows of the last replay, in its order, and each row's token is the one that
        replay sampled for it; it is taken on the device, and the entries' own token ids are ignored.
        """
        self.last_tokens = None
        if self.replays(entries):
            return self._replay(entries, reservation, draw_index, feed_back)
        if feed_back:
            raise ValueError("only a replayed step can take its tokens from the step before")
        ctx = self.build_context(entries, reservation)
        self.eager_steps += 1
        return self.model.forward(ctx, self.storage)

    def graph_for(self, n: int) -> "DecodeGraph":
        """The captured decode step of the smallest bucket that holds ``n`` rows (captured on first use)."""
        rows = next(b for b in DECODE_BUCKETS if b >= n)
        graph = self.graphs.get(rows)
        if graph is None:
            if self.graph_pool is None:
                self.graph_pool = torch.cuda.graph_pool_handle()
            graph = self.graphs[rows] = DecodeGraph(self, rows)
        return graph

    def capture_decode_graphs(self, max_rows: int) -> None:
        """Captures every bucket up to ``max_rows`` now, so that no step pays for a capture later
        (MiniServe captures its batched graphs at start-up too: miniserve/engine/graph.py:689-729)."""
        if not self.use_graphs:
            return
        for bucket in DECODE_BUCKETS:
            self.graph_for(min(bucket, max_rows))
            if bucket >= max_rows:
                break

    def _replay(self, entries, reservation, draw_index, feed_back: bool = False) -> torch.Tensor:
        n = len(entries)
        graph = self.graph_for(n)
        if feed_back and (graph is not self.last_graph or graph.live_rows != n):
            raise ValueError("the step before was not a replay of the same rows")
        if graph.copied is not None:
            graph.copied.synchronize()       # the host mirror is free once the last copy of it has run
        manager, ps = self.manager, self.manager.page_size
        limit, scratch = self.storage.num_pages, self.storage.scratch_page
        o, host = graph.offsets, graph.host_np
        if graph.live_rows != n:
            graph._fill_padding(n)
            for row in range(n, graph.rows):
                graph.row_owner[row] = None
            graph.live_rows = n
        tokens, positions, lens, slots_state = [], [], [], []
        for row, (entry, item) in enumerate(zip(entries, reservation.items)):
            token = int(entry.tokens[0])
            if entry.request_id != item.request_id or item.end - item.start != 1:
                raise ValueError(f"entry {row} does not match its reservation")
            if not 0 <= token < self.vocab_size:
                raise ValueError(f"token id {token} outside the vocabulary of {self.vocab_size}")
            if item.end > self.max_model_len:
                raise ValueError(f"request {entry.request_id!r} would reach {item.end} tokens; the limit is {self.max_model_len}")
            tokens.append(token)
            positions.append(item.start)
            lens.append(item.end)
            record = manager.requests[entry.request_id]
            slots_state.append(record.slot)
            owner = graph.row_owner[row]
            if feed_back and (owner is None or owner[0] is not record):
                raise ValueError(f"row {row} of the step before belonged to another request")
            # The row keeps what it shows only for the very same admission (a request id can come back after a
            # release, with other pages), and only as far as the pages were committed when they were written:
            # a page reserved for a step that was aborted may be another one next time.
            same = owner is not None and owner[0] is record and owner[3] == record.changes
            released_now = []
            for g in range(graph.n_groups):
                table = item.tables[g]
                if len(table) > graph.width:
                    raise ValueError("a block table is wider than the model's longest context")
                base = o[8 + 2 * g] + row * graph.width
                # committed pages that this row already shows stay; the others are checked and written
                first = owner[1][g] if same and owner[1][g] <= len(table) else 0
                released = 0
                if graph.gives_back[g]:
                    # a group behind a window or a chunk: the pages wholly before the first key that the request's next
                    # token can see went back at the last commit; the row shows the scratch page in their places
                    released = min(manager.paged_needs[g].first_needed(item.start) // ps, len(table))
                    if first > 0 and owner[2][g] <= released:
                        if released > owner[2][g]:
                            host[base + owner[2][g]:base + released] = scratch
                    else:
                        first = 0
                released_now.append(released)
                fresh = table[first:]
                if any(p != RELEASED and not 0 <= p < limit for p in fresh):
                    raise ValueError("a page lies outside the pool")
                if fresh:
                    host[base + first:base + len(table)] = [scratch if p == RELEASED else p for p in fresh]
                if first == 0:
                    host[base + len(table):base + graph.width] = scratch
                slot = int(item.slots[g][0])
                if not 0 <= slot < limit * ps:
                    raise ValueError(f"slot {slot} outside the pool")
                host[o[9 + 2 * g] + row] = slot
            graph.row_owner[row] = (record, [len(item.tables[g]) - len(item.new_pages[g]) for g in range(graph.n_groups)], released_now,
                                    record.changes)
        host[o[0]:o[0] + n] = tokens
        host[o[1]:o[1] + n] = positions
        host[o[4]:o[4] + n] = lens
        host[o[5]:o[5] + n] = slots_state
        host[o[7]:o[7] + n] = 0 if draw_index is None else list(draw_index)
        graph.meta.copy_(graph.host, non_blocking=True)
        if graph.copied is None:
            graph.copied = torch.cuda.Event()
        graph.copied.record()
        if feed_back:
            graph.meta[o[0]:o[0] + n].copy_(graph.tokens_out[:n])
        self.last_graph = graph
        graph.graph.replay()
        self.graph_replays += 1
        self.last_tokens = graph.tokens_out[:n]
        return graph.logits[:n]
