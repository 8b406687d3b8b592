"""The structural inputs of the shared-unit tests show what random ones hide (no GPU): for every listed
batch the oracle with one key, or one KV tile, lost or counted twice is out of the bounds."""

from __future__ import annotations

import pytest
import torch

from oracle import attention_tolerance
from shared_units import (PROMPTS, TILE, TREES, causal_rows, edges, equal_shares, equal_tolerance, equal_values,
                          needle_places, needle_queries, needle_reference)


def _out_of_bounds(got, want, tol):
    return bool(((got - want).abs() > tol).any())


@pytest.mark.parametrize("case", TREES + PROMPTS, ids=lambda c: f"{c['lens'][0]}x{c['dim']}")
def test_equal_weights_show_every_key(case):
    for L, n in sorted(set(zip(case["lens"], case["rows"])))[-6:]:
        if L - n < TILE:
            continue  # one tile: nothing is shared
        v = equal_values(L, 1, case["dim"], case["dtype"])
        seen = causal_rows(n, L)[-1:]
        want = equal_shares(seen, v, 1)
        tol = equal_tolerance(want, case["dtype"])
        u = torch.finfo(case["dtype"]).eps / 2
        for key in edges(L - n)[::3] + [L - n - 1]:
            for weight in (0.0, 2.0):
                w = seen.double().clone()
                w[0, key] = weight
                got = torch.einsum("nl,lhd->nhd", w, v.double()) / w.sum()
                # The kernel would round this, half a step towards the truth at worst.
                assert _out_of_bounds(got, want, tol + u * got), (L, key, weight)
        tile = seen.clone()
        tile[0, TILE:2 * TILE] = False
        assert _out_of_bounds(equal_shares(tile, v, 1), want, 2 * tol + 1e-9)


@pytest.mark.parametrize("case", [c for c in TREES + PROMPTS if len(c["lens"]) < 6], ids=lambda c: f"{c['lens'][0]}x{c['dim']}")
def test_needles_show_every_tile(case):
    g = torch.Generator().manual_seed(1)
    L, n, dim, dtype = case["lens"][0], case["rows"][0], case["dim"], case["dtype"]
    k, v = (torch.randn(L, 1, dim, generator=g).to(dtype) for _ in range(2))
    places = sorted({p for seqs in needle_places(case) for row in seqs[0] for p in row})
    assert set(edges(L - n + 1)) <= set(places)
    at = [[p] for p in places[::9] + places[-2:]]
    q = needle_queries(k, at, 1)
    seen = torch.ones(len(at), L, dtype=torch.bool)
    o, a, s = needle_reference(q, k, v, seen)
    tol = attention_tolerance(o, a, s, L, dim, dtype, v.double().abs().max().item())
    for i, (p,) in enumerate(at):
        seen[i, p // TILE * TILE:(p // TILE + 1) * TILE] = False
    got, _, _ = needle_reference(q, k, v, seen)
    worst = ((got - o).abs() / tol).amax(dim=(1, 2))
    assert worst.min().item() > 4.0, worst.min().item()
