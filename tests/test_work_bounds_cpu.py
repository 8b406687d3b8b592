"""Which sizes the attention entries take, before any GPU work (no GPU): the status says how far a call got.

A call with everything in order but its workspace ends with B200_ERR_WORKSPACE; one whose sizes
the kernels cannot count ends with B200_ERR_UNSUPPORTED before that.
"""

from __future__ import annotations

import ctypes

import pytest

from minicpm_b200 import _lib

BASE = 1 << 20  # an aligned address; nothing is read


def _prompt(total, seqs, hq, hkv, dim, total_k=None, causal=0, longest=512):
    p = _lib.PromptAttnParams(
        q=BASE, k=BASE, v=BASE, out=BASE, cu_seqlens_q=BASE, cu_seqlens_k=BASE, q_stride_t=hq * dim, q_stride_h=dim,
        k_stride_t=hkv * dim, k_stride_h=dim, v_stride_t=hkv * dim, v_stride_h=dim, out_stride_t=hq * dim, out_stride_h=dim,
        seqlen_dtype=_lib.DTYPE_I32, dtype=_lib.DTYPE_BF16, num_seqs=seqs, total_q=total,
        total_k=total if total_k is None else total_k, num_q_heads=hq, num_kv_heads=hkv, head_dim=dim, max_seqlen_k=longest,
        causal=causal, softmax_scale=0.1)
    return _lib.load().b200_prompt_attn_fwd(ctypes.byref(p), None)


@pytest.mark.parametrize(
    "total,seqs,hq,hkv,dim,total_k",
    [
        (2000 * 512, 2000, 64, 8, 128, None),
        (1100 * 1024, 2200, 32, 2, 128, None),
        (600 * 1024, 1200, 64, 8, 256, None),
        (524288, 1024, 128, 1, 128, None),
        (2 << 20, 4096, 32, 32, 128, None),
        (65536, 65536, 2, 2, 64, 1 << 20),
        (1 << 20, 1, 16, 2, 128, None),
        (16, 1, 16, 2, 128, 8 << 20),      # few rows over long keys: shared by the CTAs
        (9, 1 << 20, 8, 4, 64, 4 << 20),   # mostly empty sequences
    ],
)
@pytest.mark.parametrize("causal", [0, 1])
def test_packed_prompts_are_bounded_by_their_units_only(total, seqs, hq, hkv, dim, total_k, causal):
    assert _prompt(total, seqs, hq, hkv, dim, total_k, causal) == _lib.B200_ERR_WORKSPACE


def test_more_units_than_a_list_can_index_are_refused():
    assert _prompt(1 << 20, 1 << 20, 65535, 65535, 64) == _lib.B200_ERR_UNSUPPORTED
    assert "units" in _lib.load().b200_last_error().decode()


@pytest.mark.parametrize("cols,status", [(1 << 16, _lib.B200_ERR_WORKSPACE), (1 << 26, _lib.B200_ERR_UNSUPPORTED)])
def test_trees_are_bounded_by_their_table(cols, status):
    """64 sequences of up to 2^20 keys fit; a table of 2^30 keys a row could name more tiles than a share counts."""
    t = _lib.TreeAttnParams(
        q=BASE, k=BASE, v=BASE, out=BASE, tree_mask=BASE, block_table=BASE, cu_seqlens_q=BASE, seqused_k=BASE,
        q_stride_t=2048, q_stride_h=128, k_stride_block=4096, k_stride_tok=256, k_stride_head=128, v_stride_block=4096,
        v_stride_tok=256, v_stride_head=128, out_stride_t=2048, out_stride_h=128, mask_stride=16, block_table_stride=cols,
        mask_cols=16, block_table_cols=cols, block_table_dtype=_lib.DTYPE_I32, seqlen_dtype=_lib.DTYPE_I32,
        dtype=_lib.DTYPE_BF16, num_seqs=64, total_q=1024, num_q_heads=16, num_kv_heads=2, head_dim=128, block_size=16,
        num_blocks=100, max_seqlen_k=4096, softmax_scale=0.1)
    assert _lib.load().b200_tree_attn_fwd(ctypes.byref(t), None) == status
