"""Portions of several tokens and of several lengths behind a shared prefix, through the step function, whether or not sharing is worth it: every logit against the plain
implementation."""

from __future__ import annotations

import random

import pytest

import helpers
from test_fork_gpu import Session, runtime_of
from test_replay_gpu import check_against

import miniserve_b200  # noqa: F401
from miniserve_b200 import kernels
from miniserve_b200.engine import step as step_module

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["d", "b"])
@pytest.mark.parametrize("weighed", [True, False])
def test_portions_behind_a_prefix(request, tmp_path, monkeypatch, dtype, name, weighed):
    longest = []
    real = kernels.shared_prefix_attention
    monkeypatch.setattr(kernels, "shared_prefix_attention", lambda *a, **k: (longest.append(a[9]), real(*a, **k))[1])
    if not weighed:
        for weight in ("SHARED_KEYS_TOKEN", "SHARED_KEYS_PAIR", "SHARED_KEYS_OWN"):
            monkeypatch.setattr(step_module, weight, 0)
    folder = helpers.make_folder(tmp_path, name, seed=5)
    vocab = helpers.TINY[name]["vocab_size"]
    session = Session(runtime_of(folder, dtype, decode_execution="eager", shared_prefix_attention=True, enable_prefix_cache=False))
    rng = random.Random(7)
    some = lambda count: [rng.randrange(vocab) for _ in range(count)]
    session.admit("p")
    session.run({"p": some(200)})
    session.fork("p", ["a", "b", "c", "d"])
    session.admit("alone")
    session.run({"p": some(1), "a": some(1), "b": some(2), "c": some(5), "d": some(1), "alone": some(33)})
    session.run({"p": some(1), "a": some(70), "b": some(1), "c": some(17), "d": some(2), "alone": some(1)})
    session.run({name: some(1) for name in ("p", "a", "b", "c", "d", "alone")})
    assert (max(longest) == 70) != weighed
    check_against(request, session.got, lambda n: helpers.oracle_logits(folder, session.tokens[n]), dtype)
