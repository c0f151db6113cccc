"""Which steps read shared prefixes once, on the CPU: those of models whose attention does so, and no others leave the captured graph for it."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

import helpers
import venarax_helpers
from test_config_weights import model_for

import miniserve_b200  # noqa: F401
from miniserve_b200.cache import CacheManager
from miniserve_b200.config import resolve_architecture
from miniserve_b200.engine import step as step_module
from miniserve_b200.engine.step import StepEntry, StepFunction
from miniserve_b200.parts import DecoderModel, LayerRun, LayerSpec, ModelSpec, PartSpec

PAGE = 16


def toy(*mixers):
    """A model of one layer for every mixer."""
    rms = lambda name: PartSpec("rms", dict(name=name, size=64, eps=1e-6))
    layers = [LayerSpec(f"blocks.{i}.", mixer, PartSpec("gated_mlp", dict(hidden_size=64, intermediate_size=96)), rms("a.weight"), rms("b.weight"))
              for i, mixer in enumerate(mixers)]
    spec = ModelSpec(vocab_size=113, hidden_size=64, embedding_name="embed.weight", layers=layers, order=[LayerRun(i) for i in range(len(mixers))],
                     final_norm=rms("final.weight"), output_name=None, max_positions=4096)
    return DecoderModel(spec, torch.float32, "cpu")


def attention(**options):
    return PartSpec("attention", dict(dict(hidden_size=64, num_heads=4, num_kv_heads=2, head_dim=32, qk_norm=False, eps=1e-6, position=PartSpec("none")), **options))


SLOPES = (0.25, 0.125, 0.0625, 0.03125)
MODELS = {
    "plain": (lambda: model_for("d")[1], {0}),
    "a soft cap": (lambda: toy(attention(score_softcap=4.0)), {0}),
    "a bias by distance": (lambda: toy(attention(score_bias_slopes=SLOPES)), set()),
    "a sink": (lambda: toy(attention(sink=True)), set()),
    "a gate": (lambda: toy(attention(output_gate=True)), set()),
    "a window": (lambda: toy(attention(window=64)), set()),
    "a window in one layer": (lambda: toy(attention(window=64), attention()), {1}),
    "a bias in one layer": (lambda: toy(attention(score_bias_slopes=SLOPES), attention()), {0}),
    "other heads in one layer": (lambda: toy(attention(sink=True), attention(num_kv_heads=1)), {1}),
}


def function_of(model, shared=True):
    manager = CacheManager(model.cache_groups, PAGE, 400, 8)
    storage = SimpleNamespace(num_pages=400, scratch_page=400, scratch_slot=8)
    function = StepFunction(model, storage, manager, 4096, use_graphs=True, shared_prefixes=shared)
    manager.admit("p")
    manager.commit(manager.prepare([("p", 40 * PAGE)]))
    if all(need.keeps_all for need in manager.paged_needs) and not manager.state_needs:
        manager.fork("p", ["a", "b"])
    else:
        for name in "ab":                      # (no forks behind a window: the pages are attached by hand)
            entry = manager.admit(name)
            entry.tables, entry.length = [list(table) for table in manager.requests["p"].tables], 40 * PAGE
    return function


@pytest.mark.parametrize("name", sorted(MODELS))
def test_steps_of_a_model(monkeypatch, name):
    build, groups = MODELS[name]
    model = build()
    assert set(model.sharing_groups()) == groups
    function = function_of(model)
    entries = [StepEntry(request, [1], [0]) for request in ("p", "a", "b")]
    assert function.replays(entries)                       # (few keys: the graph)
    monkeypatch.setattr(step_module, "SHARED_KEYS_REPLAYED", 1)
    assert function.replays(entries) == (not groups)
    reservation = function.manager.prepare([(e.request_id, 1) for e in entries])
    ctx = function.build_context(entries, reservation)
    function.manager.abort(reservation)
    paged = len(function.manager.paged_needs)
    shared = ctx.shared_prefixes or [None] * paged
    assert {group for group in range(paged) if shared[group] is not None} == groups
    for group in groups:
        assert shared[group].group_start.tolist() == [0, 3] and shared[group].prefix_lens.tolist() == [40 * PAGE]


def test_without_the_option_no_step_shares():
    function = function_of(model_for("d")[1], shared=False)
    entries = [StepEntry(request, [1], [0]) for request in ("p", "a", "b")]
    reservation = function.manager.prepare([(e.request_id, 1) for e in entries])
    assert function.replays(entries) and not function.build_context(entries, reservation).shared_prefixes


def test_models_of_members_name_their_groups():
    """Mixers with several caches, states among them; Venarax's attention has sinks."""
    for raw in venarax_helpers.CONFIGS.values():
        architecture = resolve_architecture(raw)
        model = DecoderModel(architecture.build_spec(architecture.config_class.from_dict(raw)), torch.float32, "cpu")
        assert set(model.sharing_groups()) <= set(range(len(model.cache_groups)))
    inner = dict(hidden_size=64, inner=attention())
    model = toy(PartSpec("token_shift", inner))
    assert [model.run_caches[0][1].group] == sorted(model.sharing_groups())


@pytest.mark.parametrize("behind,new,alone,shares", [
    (512, [1] * 8, None, True), (512, [4] * 8, None, False), (512, [64] * 8, None, False), (512, [1] * 8, 256, False),
    (2048, [8] * 8, None, True), (2048, [128] * 4, None, False), (2048, [1] * 30, 2, True), (2048, [1] * 30, 1024, False), (2048, [1, 1], 400, False),
    (2048, [1500, 1], None, False), (3584, [1] * 30, 64, True)])
def test_prompt_portions_have_to_be_outweighed(behind, new, alone, shares):
    """Steps whose portions are long for what they share run as without the option (two query heads to a key head, eight key heads)."""
    function = function_of_heads(behind, len(new))
    entries = [StepEntry(f"r{i}", [1] * count, [count - 1]) for i, count in enumerate(new)]
    if alone is not None:
        function.manager.admit("alone")
        entries.append(StepEntry("alone", [1] * alone, [alone - 1]))
    reservation = function.manager.prepare([(e.request_id, len(e.tokens)) for e in entries])
    assert bool(function.build_context(entries, reservation).shared_prefixes) == shares


def function_of_heads(behind, count):
    model = toy(attention(num_heads=16, num_kv_heads=8, head_dim=32))
    manager = CacheManager(model.cache_groups, PAGE, 2000, 40)
    function = StepFunction(model, SimpleNamespace(num_pages=2000, scratch_page=2000, scratch_slot=40), manager, 4096, shared_prefixes=True)
    manager.admit("p")
    manager.commit(manager.prepare([("p", behind)]))
    manager.fork("p", [f"r{i}" for i in range(count)])
    return function
