"""Batches whose units several CTAs share, and values on which a lost or repeated key shows.

Random values average out: over 20000 keys a whole lost KV tile stays within a worst-case error
bound.  Two kinds of input do not average:

* equal weights: queries of 0 give every key the weight 1 (exp2(0), exact in every type), and the
  values of a sequence are one-hot, key ``j`` of ``L`` in column ``j * D // L`` (moved on by 7
  columns per KV head).  A row's output is then the share of its keys in each column.  The sums of
  weights and of values are whole numbers below 2^24, exact in fp32.
* needles: a query that is the needle's own key, at a scale that leaves the others no weight.  The
  output is the needle's value.
"""

from __future__ import annotations

import torch

from oracle.varlen_attention import attend

TILE = 128  # keys of a KV tile

BF, F16 = torch.bfloat16, torch.float16
# Trees: contexts, drafted tokens of each; prompts: keys and query rows of each sequence.
TREES = [
    dict(lens=[9016], rows=[16], hq=8, hkv=2, dim=128, dtype=BF),          # one query tile: both warpgroups on it
    dict(lens=[20003, 8], rows=[3, 3], hq=8, hkv=2, dim=64, dtype=F16),
    dict(lens=[4130], rows=[40], hq=8, hkv=2, dim=256, dtype=BF),
    dict(lens=[3040, 700], rows=[40, 33], hq=16, hkv=2, dim=128, dtype=BF),  # two query tiles, and a unit behind them
    dict(lens=[2500], rows=[130], hq=4, hkv=4, dim=64, dtype=F16),
    dict(lens=[5008, 308, 2008, 7008, 48], rows=[8] * 5, hq=16, hkv=2, dim=128, dtype=BF),
    dict(lens=[9 + (613 * i) % 1500 for i in range(70)], rows=[1 + i % 9 for i in range(70)], hq=4, hkv=1, dim=64, dtype=BF),
]
PROMPTS = [
    dict(lens=[5000], rows=[40], hq=8, hkv=2, dim=128, dtype=BF),
    dict(lens=[9001], rows=[3], hq=8, hkv=1, dim=64, dtype=F16),
    dict(lens=[3001], rows=[33], hq=4, hkv=1, dim=256, dtype=BF),
    dict(lens=[2600, 90, 1500], rows=[300, 90, 1], hq=2, hkv=2, dim=128, dtype=F16),
    dict(lens=[4100] * 75, rows=[9] * 75, hq=4, hkv=2, dim=64, dtype=BF),  # few rounds of long units
]


def equal_values(L, heads, dim, dtype):
    """One-hot values [L, heads, dim] of one sequence."""
    key = torch.arange(L)
    v = torch.zeros(L, heads, dim, dtype=dtype)
    for h in range(heads):
        v[key, h, (key * dim // L + 7 * h) % dim] = 1
    return v


def equal_shares(seen, v, hq):
    """What rows that see the keys ``seen`` [n, L] give: [n, hq, dim] in 64 bits."""
    o = torch.einsum("nl,lhd->nhd", seen.double(), v.double()) / seen.sum(dim=1).clamp_min(1)[:, None, None]
    return o.repeat_interleave(hq // v.shape[1], dim=1)


def equal_tolerance(want, dtype):
    """Weights, their sums and the sums of values are exact.  What rounds, in units of 2^-24 relative
    to non-negative terms: a piece's reciprocal, its product and the sum of two warpgroups' O (3); one
    step of the join for each of at most 148 pieces; the join's reciprocal and product (2): 160 with
    the second order.  Then the output's own rounding, half a step."""
    d = 160 * 2.0 ** -24
    return want * (torch.finfo(dtype).eps / 2 * (1 + d) + d)


def edges(L):
    """First and last key of every KV tile."""
    return sorted({p for t in range(0, L, TILE) for p in (t, min(t + TILE, L) - 1)})


def needle_queries(k, at, hq):
    """Query rows [len(at), hq, dim] that are the keys ``at`` [rows][hq] of ``k`` [L, hkv, dim]."""
    group = hq // k.shape[1]
    return torch.stack([torch.stack([k[p, h // group] for h, p in enumerate(row)]) for row in at])


def needle_places(case):
    """Rounds of places: for every row of every sequence a key per query head, so that the first and
    the last key of every tile is some row's needle.  Keys of the context only: every mask shows them."""
    todo = [edges(L - n + 1) for L, n in zip(case["lens"], case["rows"])]
    rounds = max(-(-len(e) // (n * case["hq"])) for e, n in zip(todo, case["rows"]))
    out = []
    for r in range(rounds):
        seqs = []
        for e, n in zip(todo, case["rows"]):
            first = r * n * case["hq"]
            seqs.append([[e[(first + i * case["hq"] + h) % len(e)] for h in range(case["hq"])] for i in range(n)])
        out.append(seqs)
    return out


def causal_rows(n, L):
    return torch.arange(L)[None, :] <= (L - n + torch.arange(n))[:, None]


def needle_reference(q, k, v, seen):
    return attend(q, k, v, seen, 1.0)
