"""Continuations of one cached prompt on the GPU as they are used together: a prompt is computed, forked, its continuations decode and verify drafts with
attention that reads the shared prefix once, rejected drafts are dropped, pools are compacted; every logit against the plain implementation."""

from __future__ import annotations

import random

import pytest
import torch

import helpers
from test_replay_gpu import check_against

import miniserve_b200  # noqa: F401
from miniserve_b200 import kernels
from miniserve_b200.config import EngineConfig
from miniserve_b200.engine import step as step_module
from miniserve_b200.engine.llm import LLM
from miniserve_b200.engine.runtime import build_runtime
from miniserve_b200.engine.step import StepEntry
from miniserve_b200.sampling import SamplingParams

pytestmark = pytest.mark.gpu


class Session:
    """Requests of a step function, their tokens, and every logit that was computed."""

    def __init__(self, runtime):
        self.runtime, self.manager, self.step_function = runtime, runtime.manager, runtime.step_function
        self.tokens, self.got = {}, {}

    def admit(self, name):
        self.runtime.storage.reset_slot(self.manager.admit(name).slot, 0.0, 1.0, 0, 1)
        self.tokens[name] = []

    def fork(self, name, names):
        self.step_function.fork(name, names)
        for new in names:
            self.runtime.storage.reset_slot(self.manager.requests[new].slot, 0.0, 1.0, 0, 1)
            self.tokens[new] = list(self.tokens[name])

    def run(self, tokens):
        """``{name: its next tokens}``; the logits of all of them, in order."""
        names = list(tokens)
        reservation = self.manager.prepare([(name, len(tokens[name])) for name in names])
        logits = self.step_function.run([StepEntry(name, tokens[name], list(range(len(tokens[name])))) for name in names], reservation).clone()
        self.manager.commit(reservation)
        row = 0
        for name in names:
            for token in tokens[name]:
                self.got.setdefault(name, {})[len(self.tokens[name])] = logits[row].double().cpu()
                self.tokens[name].append(token)
                row += 1
        self.manager.check_invariants()
        return logits

    def drop(self, name, length):
        self.manager.truncate(name, length)
        del self.tokens[name][length:]
        for position in [p for p in self.got.get(name, {}) if p >= length]:
            del self.got[name][position]


def runtime_of(folder, dtype, **options):
    return build_runtime(folder, EngineConfig(dtype=dtype, kv_block_size=16, num_kv_blocks=80, max_num_seqs=8, **options))


@pytest.fixture
def shared_calls(monkeypatch):
    """Counts the calls of the attention behind a shared prefix; any sharing at all is worth an eager step."""
    calls = []
    real = kernels.shared_prefix_attention
    monkeypatch.setattr(kernels, "shared_prefix_attention", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    monkeypatch.setattr(step_module, "SHARED_KEYS_REPLAYED", 1)
    return calls


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("execution", ["eager", "cuda_graph"])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("name", ["d", "b"])
def test_forks_decode_verify_and_move(request, tmp_path, shared_calls, dtype, execution, shared, name):
    folder = helpers.make_folder(tmp_path, name, seed=3)
    vocab = helpers.TINY[name]["vocab_size"]
    session = Session(runtime_of(folder, dtype, decode_execution=execution, shared_prefix_attention=shared, enable_prefix_cache=False))
    rng = random.Random(5)
    some = lambda count: [rng.randrange(vocab) for _ in range(count)]
    session.admit("filler")
    session.run({"filler": some(70)})
    session.admit("p")
    session.run({"p": some(150)})
    session.run({"p": some(43)})
    session.fork("p", ["a", "b", "c", "d"])
    names = ["p", "a", "b", "c", "d"]
    for _ in range(3):                                           # single tokens, all five
        session.run({n: some(1) for n in names})
    drafts = {n: some(count) for n, count in zip(names, (1, 4, 3, 2, 4))}
    session.run(drafts)                                          # drafted tokens, portions of several lengths
    for n, kept in zip(names, (1, 2, 0, 2, 3)):
        session.drop(n, len(session.tokens[n]) - len(drafts[n]) + kept)
    session.manager.release("filler")
    session.step_function.compact()
    allocator = session.manager.allocators[0]
    assert all(allocator.refcount(page) > 0 for page in range(allocator.used_count))
    session.run({n: some(1) for n in names})
    session.fork("b", ["e"])                                     # a fork of a fork, in the middle of a page
    session.manager.release("c")
    session.run({n: some(1) for n in ("p", "a", "b", "e", "d")})
    assert bool(shared_calls) == shared
    check_against(request, {n: rows for n, rows in session.got.items() if n != "filler"},
                  lambda n: helpers.oracle_logits(folder, session.tokens[n]), dtype)


@pytest.mark.parametrize("execution", ["eager", "cuda_graph"])
def test_drafts_give_the_tokens_of_decoding_one_by_one(tmp_path, execution):
    """Greedy drafts, some of them wrong: accepted tokens and the token behind them are what single steps choose."""
    folder = helpers.make_folder(tmp_path, "d", seed=4)
    runtime = runtime_of(folder, "float32", decode_execution=execution, shared_prefix_attention=True, enable_prefix_cache=False)
    session, rng = Session(runtime), random.Random(2)
    prompt = [rng.randrange(500) for _ in range(140)]
    session.admit("single")
    logits = session.run({"single": prompt})
    plain = [int(logits[-1].argmax())]
    while len(plain) < 30:
        plain.append(int(session.run({"single": plain[-1:]})[-1].argmax()))
    session.manager.release("single")
    session.admit("p")
    session.run({"p": prompt})
    session.fork("p", ["a", "b", "c"])
    names = ["p", "a", "b", "c"]
    done = {n: plain[:1] for n in names}
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")
    while any(len(done[n]) < 20 for n in names):
        drafts = {}
        for n in names:
            ahead = plain[len(done[n]):len(done[n]) + rng.randint(0, 4)]
            drafts[n] = [t if rng.random() < 0.7 else (t + 1) % 500 for t in ahead]
        logits = session.run({n: done[n][-1:] + drafts[n] for n in names})
        starts = [0]
        for n in names:
            starts.append(starts[-1] + len(drafts[n]))
        accepted, token = torch.empty(4, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
        flat = ints(sum((drafts[n] for n in names), []))
        kernels.verify_drafts(logits, flat, ints(starts), torch.rand(len(flat), device="cuda"), torch.empty(4, 500, device="cuda").exponential_(),
                              accepted, token, records=runtime.storage.sampling_records,
                              slot_of_request=ints([session.manager.requests[n].slot for n in names]))
        for n, kept, following in zip(names, accepted.tolist(), token.tolist()):
            session.drop(n, len(session.tokens[n]) - len(drafts[n]) + kept)
            done[n] = done[n] + drafts[n][:kept] + [following]
    for n in names:
        assert done[n] == plain[:len(done[n])]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_replayed_steps_see_what_a_truncation_or_a_move_changed(request, tmp_path, dtype):
    """A request drops pages that another one then takes, and comes back to the same number of pages with others; then all pages move.  The captured steps'
    copy of its table must not show the old ones."""
    folder = helpers.make_folder(tmp_path, "d", seed=6)
    session = Session(runtime_of(folder, dtype, decode_execution="cuda_graph", enable_prefix_cache=False))
    rng = random.Random(8)
    some = lambda count: [rng.randrange(500) for _ in range(count)]
    for n, count in (("a", 60), ("b", 20)):
        session.admit(n)
        session.run({n: some(count)})
    for _ in range(8):
        session.run({"a": some(1), "b": some(1)})
    session.drop("a", 17)
    session.run({"b": some(50)})                                  # takes the pages that a gave back
    session.run({"a": some(48)})
    for _ in range(3):
        session.run({"a": some(1), "b": some(1)})
    session.drop("b", 5)
    session.step_function.compact()
    for _ in range(14):
        session.run({"a": some(1), "b": some(1)})
    check_against(request, session.got, lambda n: helpers.oracle_logits(folder, session.tokens[n]), dtype)


@pytest.mark.parametrize("execution", ["eager", "cuda_graph"])
def test_generation_with_a_shared_prompt(tmp_path, shared_calls, execution):
    """Requests whose prompts start alike, through the engine: the tokens are those without the option."""
    folder = helpers.make_folder(tmp_path, "d", seed=9)
    rng = random.Random(1)
    start = [rng.randrange(500) for _ in range(300)]
    prompts = [start + [rng.randrange(500) for _ in range(n)] for n in (3, 17, 1, 40)]
    params = [SamplingParams(max_new_tokens=12), SamplingParams(max_new_tokens=9, temperature=0.8, top_p=0.9, seed=3), SamplingParams(max_new_tokens=20),
              SamplingParams(max_new_tokens=5)]
    results = []
    for shared in (False, True):
        llm = LLM(str(folder), dtype="float32", max_num_seqs=4, num_kv_blocks=120, kv_block_size=16, decode_execution=execution,
                  shared_prefix_attention=shared)
        llm.generate([start], SamplingParams(max_new_tokens=1))          # (fills the prefix cache)
        assert not shared_calls or shared
        results.append([r.token_ids for r in llm.generate(prompts, params)])
    assert shared_calls and results[0] == results[1]
