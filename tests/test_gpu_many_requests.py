"""Packed batches whose sizes, taken for one sequence, would be more work than a tick counter holds (GPU)."""

from __future__ import annotations

import pytest
import torch

from minicpm_b200 import _lib, prompt_attention
from oracle import attention_tolerance

pytestmark = pytest.mark.gpu


def test_a_million_tokens_in_short_requests():
    """65536 requests of one query row over 16 keys: 131072 units, 1 M rows of K and V."""
    n, keys, heads, dim, dtype = 65536, 16, 2, 64, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(rows, heads, dim, generator=g, device="cuda").to(dtype) for rows in (n, n * keys, n * keys))
    out = torch.full_like(q, float("nan"))
    cu = torch.arange(n + 1, device="cuda", dtype=torch.int32)
    prompt_attention(q, k, v, out, cu, 1, 0.3, cu_seqlens_k=cu * keys, max_seqlen_k=keys)
    assert _lib.device_error() == _lib.DEVERR_NONE
    for at in range(0, n, 8192):
        rows, kv = slice(at, at + 8192), slice(at * keys, (at + 8192) * keys)
        kd, vd = (t[kv].double().view(-1, keys, heads, dim) for t in (k, v))
        x = torch.einsum("nhd,nkhd->nhk", q[rows].double(), kd) * 0.3
        s = torch.einsum("nhd,nkhd->nhk", q[rows].double().abs(), kd.abs()).amax(dim=-1) * 0.3
        p = torch.softmax(x, dim=-1)
        o, a = torch.einsum("nhk,nkhd->nhd", p, vd), torch.einsum("nhk,nkhd->nhd", p, vd.abs())
        tol = attention_tolerance(o, a, s, keys, dim, dtype, vd.abs().max().item())
        assert ((out[rows].double() - o).abs() <= tol).all()
