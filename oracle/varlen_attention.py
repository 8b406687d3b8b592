"""64-bit CPU restatement of the packed prompt attention and the draft-tree attention.

TEST INFRASTRUCTURE ONLY (never shipped).  No counterpart in the
reference: the operators are defined by their formulas.

Beside the result, :func:`attend` gives what an error bound needs: ``A = sum_j
p_ij |v_j|`` and the largest ``scale * sum_d |q_id k_jd|`` of each row.
"""

from __future__ import annotations

from typing import Sequence

import torch


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor, scale: float):
    """One sequence: ``q [n, Hq, D]``, ``k``/``v [L, KH, D]``, ``seen [n, L]``; returns ``(o, A, s)`` in float64.

    A row that sees no key is 0.  Keys no row sees may hold anything.
    """
    n, hq, d = q.shape
    group = hq // k.shape[1]
    used = seen.any(dim=0)
    k = torch.where(used[:, None, None], k.double(), 0.0).repeat_interleave(group, dim=1)
    v = torch.where(used[:, None, None], v.double(), 0.0).repeat_interleave(group, dim=1)
    x = torch.einsum("nhd,lhd->hnl", q.double(), k) * scale
    s = torch.einsum("nhd,lhd->hnl", q.double().abs(), k.abs()).amax(dim=-1) * scale if k.shape[0] else torch.zeros(hq, n)
    x = x.masked_fill(~seen[None], float("-inf"))
    has = seen.any(dim=1)
    p = torch.softmax(x, dim=-1) if k.shape[0] else x
    p = torch.where(has[None, :, None], p, torch.zeros_like(p))
    return torch.einsum("hnl,lhd->nhd", p, v), torch.einsum("hnl,lhd->nhd", p, v.abs()), s.transpose(0, 1)


def _collect(parts, total, q):
    o, a = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    s = torch.zeros(q.shape[:2], dtype=torch.float64)
    for begin, (x, y, z) in parts:
        o[begin:begin + x.shape[0]], a[begin:begin + x.shape[0]], s[begin:begin + x.shape[0]] = x, y, z
    return o, a, s


def prompt_attention_reference(q, k, v, cu_q: Sequence[int], cu_k: Sequence[int], scale: float, causal: bool):
    """Packed sequences over plain rows: ``(o, A, s)`` as :func:`attend`."""
    parts = []
    for b in range(len(cu_q) - 1):
        n, L = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        seen = torch.ones(n, L, dtype=torch.bool)
        if causal:
            seen = torch.arange(L)[None, :] <= (L - n + torch.arange(n))[:, None]
        parts.append((cu_q[b], attend(q[cu_q[b]:cu_q[b + 1]], k[cu_k[b]:cu_k[b + 1]], v[cu_k[b]:cu_k[b + 1]], seen, scale)))
    return _collect(parts, cu_q[-1], q)


def tree_attention_reference(q, k_cache, v_cache, tree_mask, block_table, lens: Sequence[int], cu_q: Sequence[int],
                             scale: float):
    """Drafted tokens over a paged cache: ``(o, A, s)`` as :func:`attend`."""
    parts = []
    page = k_cache.shape[1]
    for b, L in enumerate(lens):
        n = cu_q[b + 1] - cu_q[b]
        pages = block_table[b, :-(-L // page)].long()
        k, v = (c[pages].reshape(-1, c.shape[2], c.shape[3])[:L] for c in (k_cache, v_cache))
        key = torch.arange(L)[None, :] - (L - n)  # drafted index of each key, negative in the context
        seen = (key < 0).expand(n, L).clone()
        for i in range(n):
            for j in range(max(0, n - L), min(n, tree_mask.shape[1])):
                seen[i, L - n + j] = bool(tree_mask[cu_q[b] + i, j])
        parts.append((cu_q[b], attend(q[cu_q[b]:cu_q[b + 1]], k, v, seen, scale)))
    return _collect(parts, cu_q[-1], q)


def attention_tolerance(o: torch.Tensor, a: torch.Tensor, s: torch.Tensor, keys: int, dim: int, dtype: torch.dtype,
                        v_max: float):
    """Largest error the kernel may show against 64 bits, element by element.

    Two roundings to the element type, half a step ``u`` each: the softmax weight of every
    key (at most ``u A`` in the sum) and the output (``u (|o| + error)``).  The rest is fp32:
    a score is a sum of ``dim`` products (relative to their absolute sum ``s``: ``dim`` 2^-23),
    which enters a weight as its exponent, above and below the fraction; the weights' sum and
    the weighted sum of ``keys`` terms each err by ``keys`` 2^-23; 2^-20 covers the exponential.
    f16 weights below 2^-14 round to steps of 2^-24 (the largest weight of a row is at least 1
    and its sum too): half a step of each of ``keys`` values up to ``v_max``.
    """
    u = torch.finfo(dtype).eps / 2
    fp32 = 2.0 * s[..., None] * dim * 2.0 ** -23 + 2.0 * keys * 2.0 ** -23 + 2.0 ** -20
    err = a * (u + fp32)
    if dtype == torch.float16:
        err = err + keys * 2.0 ** -25 * v_max
    return err + u * (o.abs() + err) + 1e-30
