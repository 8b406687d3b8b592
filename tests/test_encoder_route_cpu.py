"""Which encoder batches of the service take the sm_100a kernel, and metadata of other makers (no GPU)."""

from __future__ import annotations

import sys
from types import ModuleType, SimpleNamespace

import pytest
import torch

from minicpm_b200 import service

BF = torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    """Both flags set; both kernels replaced by a record of the call."""
    seen = []
    module = ModuleType("vllm.v1.attention.ops.triton_prefill_attention")
    module.context_attention_fwd = lambda **kw: seen.append(("vllm", kw))
    for name in ("vllm", "vllm.v1", "vllm.v1.attention", "vllm.v1.attention.ops"):
        monkeypatch.setitem(sys.modules, name, ModuleType(name))
    monkeypatch.setitem(sys.modules, module.__name__, module)
    monkeypatch.setattr(service, "prompt_attention", lambda *a, **kw: seen.append(("prompt", a)))
    monkeypatch.setenv("ILUVATAR_USE_OPTIMIZED", "1")
    monkeypatch.setenv("ILUVATAR_SPLIT_KV", "1")
    return seen


def _meta(n):
    return SimpleNamespace(use_cascade=False, num_actual_tokens=n, query_start_loc=torch.tensor([0, n], dtype=torch.int32),
                           max_query_len=n, seq_lens=torch.tensor([n], dtype=torch.int32))


def _rows(n, heads, dim=128, shift=0, pad=0):
    """[n, heads, dim] whose first element lies `shift` elements, and whose rows `pad` elements, off the packed place."""
    buf = torch.zeros(n * (heads * dim + pad) + shift + 16, dtype=BF)
    return buf[shift:].as_strided((n, heads, dim), (heads * dim + pad, dim, 1))


def _route(calls, query, key, value, output, scale=0.1):
    impl = service.IluvatarAttentionImpl(query.shape[1], query.shape[2], scale, key.shape[1], None, None, "auto",
                                         attn_type=service.AttentionType.ENCODER_ONLY)
    impl.forward(SimpleNamespace(), query, key, value, torch.zeros(0), _meta(query.shape[0]), output)
    assert len(calls) == 1
    return calls.pop()[0]


def test_plain_and_strided_batches_take_the_kernel(calls):
    for pad in (0, 8, 2560):  # views of a fused q/k/v projection among them
        q, k, v, o = _rows(9, 16, pad=pad), _rows(9, 2, pad=pad), _rows(9, 2, pad=pad), _rows(9, 16, pad=pad)
        assert _route(calls, q, k, v, o) == "prompt"
    one = [_rows(1, h, shift=8).as_strided((1, h, 128), (3, 128, 1), 8) for h in (16, 2, 2, 16)]
    assert _route(calls, *one) == "prompt"  # a dimension of one element takes any stride


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("shift,pad", [(1, 0), (4, 0), (0, 4), (0, 1)])
def test_rows_off_the_kernels_grid_go_to_vllm(calls, which, shift, pad):
    t = [_rows(9, h) for h in (16, 2, 2, 16)]
    t[which] = _rows(9, t[which].shape[1], shift=shift, pad=pad)
    assert _route(calls, *t) == "vllm"


def test_dimensions_that_are_not_contiguous_go_to_vllm(calls):
    q, k, v, o = (_rows(9, h) for h in (16, 2, 2, 16))
    wide = torch.zeros(9, 2, 256, dtype=BF)[:, :, ::2]
    assert _route(calls, q, wide, v, o) == "vllm"
    assert _route(calls, q, k, wide, o) == "vllm"


@pytest.mark.parametrize("scale", [0.0, -0.5])
def test_scales_that_the_kernel_refuses_go_to_vllm(calls, scale):
    assert _route(calls, *(_rows(9, h) for h in (16, 2, 2, 16)), scale=scale) == "vllm"
