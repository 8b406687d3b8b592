"""int64 ends of sequences past int32, on units that several CTAs share (GPU): the attention kernel
and the join behind it read the same rows."""

from __future__ import annotations

import pytest
import torch

from minicpm_b200 import _lib, prompt_attention
from test_gpu_tree_attention import Batch

pytestmark = pytest.mark.gpu

# Every pair clips to the rows [0, 8); cut to 32 bits the second and third name fewer.
ENDS = [(0, 8), (0, (1 << 32) + 5), (-(1 << 40) + 3, 8), (-1, 1 << 40)]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("ends", ENDS)
def test_prompt_rows_past_int32(ends, dim):
    g = torch.Generator().manual_seed(dim)
    q, k, v = (torch.randn(n, h, dim, generator=g).to(torch.bfloat16).cuda() for n, h in ((8, 8), (5000, 2), (5000, 2)))
    cu_k = torch.tensor([0, 5000], device="cuda")

    def run(cu, keys):
        out = torch.full_like(q, float("nan"))
        return prompt_attention(q, k, v, out, torch.tensor(cu, device="cuda"), 8, dim ** -0.5, cu_seqlens_k=keys,
                                max_seqlen_k=5000)

    want = run((0, 8), cu_k)
    assert torch.isfinite(want.float()).all()
    assert torch.equal(run(ends, cu_k), want)
    assert torch.equal(run(ends, torch.tensor([-(1 << 33), (1 << 32) + 77], device="cuda")), want)
    assert _lib.device_error() == _lib.DEVERR_NONE


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("ends", ENDS)
def test_tree_rows_past_int32(ends, dim):
    b = Batch([5000], [8], hq=8, dim=dim, seed=dim)
    wide = dict(seqused_k=torch.tensor(b.lens).cuda())
    want = b.run(cu_seqlens_q=b.cu.long().cuda(), **wide)
    b.check(want)
    assert torch.equal(b.run(cu_seqlens_q=torch.tensor(ends).cuda(), **wide), want)
    assert _lib.device_error() == _lib.DEVERR_NONE
