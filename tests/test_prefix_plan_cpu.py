"""The plan of the attention behind shared prefixes for bounds of every kind, on the CPU (the library answers without a GPU)."""

from __future__ import annotations

import itertools

import miniserve_b200  # noqa: F401
from miniserve_b200 import kernels


def test_every_bound_has_a_plan():
    for code, aligned, d, (n_q, n_kv), page in itertools.product((0, 1), (0, 1), (7, 40, 64, 128, 512), ((1, 1), (8, 2), (256, 1)), (1, 16, 24, 128)):
        for groups, group_tokens, prefix, requests, tokens, suffix in itertools.product((0, 1, 3), (0, 1, 5000), (0, 1, 100000), (0, 1, 300), (0, 1, 9000), (0, 1, 100000)):
            plan = kernels.library().ms_prefix_attention_plan(code, aligned, d, n_q, n_kv, page, groups, group_tokens, prefix, requests, tokens, suffix)
            assert plan >> 16 in (0, 1) and 0 <= plan >> 8 & 255 <= 64 and 1 <= plan & 255 <= 64
            assert (plan >> 8 & 255 > 0) == (prefix > 0)
