"""Units that several CTAs share (GPU): every key counts once, wherever a share ends.  The inputs
are those of ``shared_units``, on which a single lost or repeated key shows."""

from __future__ import annotations

import pytest
import torch

from minicpm_b200 import _lib, prompt_attention
from oracle import attention_tolerance
from shared_units import (PROMPTS, TREES, causal_rows, equal_shares, equal_tolerance, equal_values, needle_places,
                          needle_queries, needle_reference)
from test_gpu_tree_attention import Batch

pytestmark = pytest.mark.gpu


def _ids(case):
    return f"{len(case['lens'])}x{case['lens'][0]}x{case['dim']}"


def _cu(lens):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)


def _within(out, want, tol, what):
    d = (out.cpu().double() - want).abs()
    assert torch.isfinite(d).all(), what
    assert (d <= tol).all(), f"{what}: {(d / tol.clamp_min(1e-30)).max().item():.2f} of the bound"


def _tree(case, page=16):
    b = Batch([L - n for L, n in zip(case["lens"], case["rows"])], case["rows"], hq=case["hq"], hkv=case["hkv"],
              dim=case["dim"], dtype=case["dtype"], page=page, seed=len(case["lens"]))
    width = max(case["rows"])
    b.mask = torch.cat([torch.tril(torch.ones(n, width, dtype=torch.bool)) for n in case["rows"]])
    return b


def _put(b, row, part, values):
    """Rows of a sequence to their places in the cache (part 0: keys, 1: values)."""
    pos = torch.arange(values.shape[0])
    b.cache[b.table[row, pos // b.page].long(), part, pos % b.page] = values


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("case", TREES, ids=_ids)
def test_trees_with_equal_weights(case, page):
    b = _tree(case, page)
    b.q.zero_()
    values = [equal_values(L, case["hkv"], case["dim"], case["dtype"]) for L in b.lens]
    for row, v in enumerate(values):
        _put(b, row, 1, v)
    out = b.run()
    for row, (L, n, v) in enumerate(zip(b.lens, b.nodes, values)):
        want = equal_shares(causal_rows(n, L), v, case["hq"])
        _within(out[b.cu[row]:b.cu[row + 1]], want, equal_tolerance(want, case["dtype"]), f"sequence {row}")
    assert _lib.device_error() == _lib.DEVERR_NONE


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", PROMPTS, ids=_ids)
def test_prompts_with_equal_weights(case, causal):
    ql, kl, dim, dtype = case["rows"], case["lens"], case["dim"], case["dtype"]
    values = [equal_values(L, case["hkv"], dim, dtype) for L in kl]
    q = torch.zeros(sum(ql), case["hq"], dim, dtype=dtype, device="cuda")
    k = torch.randn(sum(kl), case["hkv"], dim, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    out = torch.full_like(q, float("nan"))
    cu = _cu(ql)
    prompt_attention(q, k, torch.cat(values).cuda(), out, cu.cuda(), max(ql), 0.1, causal=causal, cu_seqlens_k=_cu(kl).cuda(),
                     max_seqlen_k=max(kl))
    for row, (n, L, v) in enumerate(zip(ql, kl, values)):
        seen = causal_rows(n, L) if causal else torch.ones(n, L, dtype=torch.bool)
        want = equal_shares(seen, v, case["hq"])
        _within(out[cu[row]:cu[row + 1]], want, equal_tolerance(want, dtype), f"sequence {row}")
    assert _lib.device_error() == _lib.DEVERR_NONE


SINGLE = [c for c in TREES if len(c["lens"]) < 6]


@pytest.mark.parametrize("case", SINGLE, ids=_ids)
def test_trees_find_their_needles(case):
    b = _tree(case)
    b.scale = 1.0
    cache = b.cache.cuda()
    rows = []
    for row, L in enumerate(b.lens):
        pages = b.table[row, :-(-L // b.page)].long()
        rows.append([b.cache[pages, part].reshape(-1, case["hkv"], case["dim"])[:L] for part in (0, 1)])
    v_max = b.cache.double().abs().max().item()
    for places in needle_places(case):
        b.q = torch.cat([needle_queries(k, at, case["hq"]) for (k, _), at in zip(rows, places)])
        out = b.run(cache=cache)
        for row, ((k, v), L, n) in enumerate(zip(rows, b.lens, b.nodes)):
            at = slice(int(b.cu[row]), int(b.cu[row + 1]))
            o, a, s = needle_reference(b.q[at], k, v, causal_rows(n, L))
            _within(out[at], o, attention_tolerance(o, a, s, L, case["dim"], case["dtype"], v_max), f"sequence {row}")


@pytest.mark.parametrize("case", [c for c in PROMPTS if len(c["lens"]) < 6], ids=_ids)
def test_prompts_find_their_needles(case):
    ql, kl, dim, dtype = case["rows"], case["lens"], case["dim"], case["dtype"]
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(sum(kl), case["hkv"], dim, generator=g).to(dtype) for _ in range(2))
    cu, ck = _cu(ql), _cu(kl)
    seqs = [slice(int(ck[i]), int(ck[i + 1])) for i in range(len(kl))]
    args = (k.cuda(), v.cuda())
    for places in needle_places(case):
        q = torch.cat([needle_queries(k[s], at, case["hq"]) for s, at in zip(seqs, places)])
        out = torch.full(q.shape, float("nan"), dtype=dtype, device="cuda")
        prompt_attention(q.cuda(), *args, out, cu.cuda(), max(ql), 1.0, causal=True, cu_seqlens_k=ck.cuda(),
                         max_seqlen_k=max(kl))
        for row, (s, n, L) in enumerate(zip(seqs, ql, kl)):
            at = slice(int(cu[row]), int(cu[row + 1]))
            o, a, x = needle_reference(q[at], k[s], v[s], causal_rows(n, L))
            _within(out[at], o, attention_tolerance(o, a, x, L, dim, dtype, v.double().abs().max().item()), f"sequence {row}")
    assert _lib.device_error() == _lib.DEVERR_NONE
