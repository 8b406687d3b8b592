"""The largest softmax_scale of prompt and tree attention: refused where its base-2 form is not finite,
and right up to there."""

from __future__ import annotations

import ctypes

import pytest
import torch

from minicpm_b200 import _lib, paged_tree_attention, prompt_attention
from test_gpu_tree_attention import Batch
from test_serving_operators_cpu import _prompt, _tree


@pytest.mark.parametrize("scale", [2.1e38, 2.4e38, 2.9e38, 3.4e38])
def test_scales_past_the_largest_are_refused(scale):
    with pytest.raises(ValueError, match="softmax_scale"):
        prompt_attention(**_prompt(softmax_scale=scale))
    with pytest.raises(ValueError, match="softmax_scale"):
        paged_tree_attention(**_tree(softmax_scale=scale))
    p = _lib.PromptAttnParams(dtype=_lib.DTYPE_BF16, num_q_heads=4, num_kv_heads=2, head_dim=64, seqlen_dtype=_lib.DTYPE_I32,
                              softmax_scale=scale)
    assert _lib.load().b200_prompt_attn_fwd(ctypes.byref(p), None) == _lib.B200_ERR_INVALID
    p.softmax_scale = 2.0e38
    assert _lib.load().b200_prompt_attn_fwd(ctypes.byref(p), None) == _lib.B200_OK  # no tokens


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0e38, 1e-44])
def test_scores_of_zero_at_the_ends_of_the_range(scale):
    """Queries of 0: every visible key weighs the same at any scale."""
    b = Batch([300], [4], hq=8, hkv=2, dim=64, seed=1)
    b.q.zero_()
    b.scale = scale
    b.check(b.run())
    q, v = torch.zeros(130, 4, 64, dtype=torch.float16, device="cuda"), torch.ones(130, 2, 64, dtype=torch.float16, device="cuda")
    out = torch.empty_like(q)
    prompt_attention(q, torch.randn_like(v), v, out, torch.tensor([0, 130], device="cuda"), 130, scale)
    assert (out == 1).all() and _lib.device_error() == _lib.DEVERR_NONE
