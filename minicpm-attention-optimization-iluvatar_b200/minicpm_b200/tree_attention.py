"""Attention of drafted token trees over a paged cache on sm_100a.

Speculative decoding verifies the drafted tokens of every sequence in one pass:
their K/V rows are written to the cache behind the context (as any new token's),
and each token attends to the context and to its own ancestors in the tree.  One
call of ``b200_tree_attn_fwd``: the tcgen05 attention kernel in its form for trees, whose
CTAs divide all keys among themselves, and a join of the units that several of them
share, on the current CUDA stream without a host synchronisation.  No counterpart in the reference.
:func:`minicpm_b200.kv_pages.keep_accepted_tokens` then moves the accepted path
together in the cache.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

_INDEX_TYPES = (torch.int32, torch.int64)
_ELEMENT_TYPES = (torch.bfloat16, torch.float16)
_MASK_TYPES = (torch.bool, torch.uint8)


def paged_tree_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    tree_mask: torch.Tensor,
    block_table: torch.Tensor,
    seqused_k: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    max_seqlen_q: int,
    max_seqlen_k: int,
    softmax_scale: float,
) -> torch.Tensor:
    """Attend the drafted tokens of every sequence to its context and their tree; returns ``out``.

    ``q``/``out`` ``[T, Hq, D]``, the caches ``k``/``v`` ``[num_blocks, block_size, KH, D]``,
    ``block_table``, ``seqused_k`` and ``cu_seqlens_q`` as in
    :func:`~minicpm_b200.paged_split_kv_attention`.  The last ``n = cu_seqlens_q[b + 1] -
    cu_seqlens_q[b]`` of the ``seqused_k[b]`` cached tokens of sequence ``b`` are its
    drafted ones.  ``tree_mask`` ``[T, W]`` (bool or uint8, W >= ``max_seqlen_q``): row ``t``
    sees drafted token ``j`` of its sequence iff ``tree_mask[t, j]``; it sees every token of
    the context.  A drafted token usually sees itself and its ancestors, but any mask goes;
    a row that sees nothing is 0.  Rows of ``out`` that belong to no sequence are left as
    they were.  Cached keys and values that some row sees must be finite; drafted tokens that
    no row sees (slots of a padded draft) and those past a sequence's length may hold
    anything.  A lower-triangular mask gives causal attention; one token per sequence with
    ``tree_mask[t, 0]`` set is a decode step.

    The batch's units of work (one per sequence and KV head at least) times the 128-key tiles
    of a full row of the block table stay below 2^30, else ``RuntimeError``.
    """
    if q.ndim != 3 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("expected q=[T,H,D] and k/v=[blocks,block,kv_heads,D]")
    q_shape, k_shape = q.shape, k.shape
    if out.shape != q_shape or k_shape != v.shape:
        raise ValueError("out must match q and k/v must have identical shapes")
    dev = q.device
    if not (dev == k.device == v.device == out.device == tree_mask.device == block_table.device == seqused_k.device
            == cu_seqlens_q.device):
        raise ValueError("all tensors must be on the same device")
    table_dtype, len_dtype = block_table.dtype, seqused_k.dtype
    if block_table.ndim != 2 or table_dtype not in _INDEX_TYPES:
        raise ValueError("block_table must contain integer physical block ids")
    if cu_seqlens_q.ndim != 1 or seqused_k.ndim != 1:
        raise ValueError("cu_seqlens_q and seqused_k must be one-dimensional")
    num_seqs = seqused_k.shape[0]
    table_rows, table_cols = block_table.shape
    if cu_seqlens_q.shape[0] != num_seqs + 1:
        raise ValueError("cu_seqlens_q must contain one entry per request plus one")
    if table_rows != num_seqs:
        raise ValueError("block_table and seqused_k must have the same request count")
    if cu_seqlens_q.dtype != len_dtype or len_dtype not in _INDEX_TYPES:
        raise ValueError("cu_seqlens_q and seqused_k must be int32 or int64 of one dtype")
    total_q, hq, head_dim = q_shape
    num_blocks, block_size, hkv, dk = k_shape
    if (dk != head_dim or head_dim not in (64, 128, 256) or hkv == 0 or hq == 0 or hq % hkv or block_size <= 0
            or block_size % 16):
        raise ValueError("unsupported head shape for tree attention")
    if tree_mask.ndim != 2 or tree_mask.dtype not in _MASK_TYPES or tree_mask.shape[0] != total_q:
        raise ValueError("tree_mask must be bool or uint8 with one row per query token")
    mask_cols = tree_mask.shape[1]
    if mask_cols < max_seqlen_q:
        raise ValueError("tree_mask must have a column for each of the max_seqlen_q drafted tokens")
    if not 0.0 < softmax_scale <= _lib.MAX_SOFTMAX_SCALE:
        raise ValueError("softmax_scale must be positive and at most 2e38")
    if not q.is_cuda:
        raise RuntimeError("paged_tree_attention runs on CUDA tensors only (no CPU path)")
    dtype = q.dtype
    if dtype not in _ELEMENT_TYPES or not (dtype == k.dtype == v.dtype == out.dtype):
        raise RuntimeError("the sm_100a kernel takes bf16 or f16 q/k/v/out of one dtype")
    (qt, qh, qd), (kb, kt, kh, kd), (vb, vt, vh, vd), (ot, oh, od) = q.stride(), k.stride(), v.stride(), out.stride()
    if not (qd == kd == vd == od == 1):
        raise RuntimeError("the head dimension of q, k, v and out must be contiguous")
    if num_blocks == 0 or table_cols == 0:
        raise ValueError("the cache and the block table must have at least one page")
    if total_q == 0 or num_seqs == 0:
        return out
    # A dimension of one element may carry any stride: it counts as packed.
    if hq == 1:
        qh = oh = head_dim
    if hkv == 1:
        kh = vh = head_dim
    if total_q == 1:
        qt, ot = hq * qh, hq * oh
    if num_blocks == 1:
        kb, vb = block_size * kt, block_size * vt
    mask_stride, mask_step = tree_mask.stride()
    if mask_step != 1:
        tree_mask = tree_mask.contiguous()
        mask_stride = mask_cols
    table_stride, table_step = block_table.stride()
    if table_step != 1:
        block_table = block_table.contiguous()
        table_stride = table_cols
    if not (cu_seqlens_q.is_contiguous() and seqused_k.is_contiguous()):
        cu_seqlens_q, seqused_k = cu_seqlens_q.contiguous(), seqused_k.contiguous()
    max_seqlen_k = int(max_seqlen_k)
    lib = _lib.load()
    with _lib.on_device(dev):
        nbytes = _lib.varlen_workspace_bytes(dev.index, total_q, num_seqs, hq, hkv, head_dim, max_seqlen_k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p = _lib.TreeAttnParams(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), tree_mask.data_ptr(), block_table.data_ptr(),
            cu_seqlens_q.data_ptr(), seqused_k.data_ptr(), qt, qh, kb, kt, kh, vb, vt, vh, ot, oh, mask_stride, table_stride,
            mask_cols, table_cols, _lib.dtype_code(table_dtype), _lib.dtype_code(len_dtype), _lib.dtype_code(dtype),
            num_seqs, total_q, hq, hkv, head_dim, block_size, num_blocks, max_seqlen_k, softmax_scale, ws.data_ptr(), nbytes,
        )
        _lib.check(lib.b200_tree_attn_fwd(ctypes.byref(p), _lib.current_stream(dev)), "paged_tree_attention")
    return out


__all__ = ["paged_tree_attention"]
