"""Metadata that knows nothing of draft trees runs as it always did (no GPU)."""

from __future__ import annotations

from types import SimpleNamespace

import torch

from minicpm_b200 import service

BF = torch.bfloat16


def test_metadata_of_another_maker_needs_no_tree_mask(monkeypatch):
    calls = []
    monkeypatch.setattr(service, "unified_attention_optimized", lambda **kw: calls.append(kw))
    monkeypatch.setenv("ILUVATAR_USE_OPTIMIZED", "1")
    monkeypatch.setenv("ILUVATAR_SPLIT_KV", "1")
    meta = SimpleNamespace(  # the fields that the layer read before it knew of trees
        use_cascade=False, num_actual_tokens=9, query_start_loc=torch.tensor([0, 9], dtype=torch.int32), max_query_len=9,
        seq_lens=torch.tensor([64], dtype=torch.int32), max_seq_len=64, causal=True, block_table=torch.zeros(1, 4),
        seq_threshold_3D=None, num_par_softmax_segments=None, softmax_segm_output=None, softmax_segm_max=None,
        softmax_segm_expsum=None, mm_prefix_range_tensor=None)
    impl = service.IluvatarAttentionImpl(16, 128, 0.1, 2, None, None, "auto")
    q = torch.zeros(9, 16, 128, dtype=BF)
    impl.forward(SimpleNamespace(), q, q, q, torch.zeros(4, 2, 16, 2, 128, dtype=BF), meta, torch.empty_like(q))
    assert len(calls) == 1 and calls[0].get("tree_mask") is None
