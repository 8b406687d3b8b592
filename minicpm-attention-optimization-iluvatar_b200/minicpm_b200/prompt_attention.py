"""Attention of packed prompts over plain K/V rows on sm_100a.

The first pass over a prompt, an encoder batch or an embedding batch needs no
cache: sequences of different lengths lie one after the other in ``q``, ``k`` and
``v`` (``cu_seqlens``), query heads share KV heads (any ratio up to 128) and a row
sees its sequence causally or whole.  One call of ``b200_prompt_attn_fwd``: for
batches that fill the GPU a device-side work list and the tcgen05 attention kernel in
its form for plain rows; else that kernel alone, whose CTAs divide all keys among
themselves, and a join of the units that several of them share.  All on the current
CUDA stream without a host synchronisation.  No counterpart in the
reference, whose service sends encoder batches to vLLM
(``integration/vllm-plugin-FL-split-kv.patch:785-813``).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib

_INDEX_TYPES = (torch.int32, torch.int64)
_ELEMENT_TYPES = (torch.bfloat16, torch.float16)


def prompt_layout_supported(*rows: torch.Tensor, softmax_scale: float) -> bool:
    """Whether the kernel can address these ``[T, H, D]`` tensors, and takes the scale.

    For callers that have another kernel for such a call; types and head shapes are
    :func:`~minicpm_b200.split_kv_paged.kernel_supports`'s part.
    """
    for t in rows:
        if t.ndim != 3:
            return False
        tokens, heads, _ = t.shape
        st, sh, sd = t.stride()
        if sd != 1 or t.data_ptr() % 16 or (heads > 1 and sh % 8) or (tokens > 1 and st % 8):
            return False
    return 0.0 < softmax_scale <= _lib.MAX_SOFTMAX_SCALE


def prompt_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    max_seqlen_q: int,
    softmax_scale: float,
    causal: bool = True,
    cu_seqlens_k: Optional[torch.Tensor] = None,
    max_seqlen_k: Optional[int] = None,
) -> torch.Tensor:
    """``out[i] = softmax(softmax_scale * q[i] . k[j]) v[j]`` within each sequence; returns ``out``.

    ``q``/``out`` ``[total_q, Hq, D]``, ``k``/``v`` ``[total_k, KH, D]`` (bf16 or f16,
    D 64, 128 or 256, D contiguous, other strides multiples of 8 elements, 16-byte
    aligned).  Sequence ``b`` owns the rows ``cu_seqlens_q[b]:cu_seqlens_q[b + 1]`` of
    ``q`` and ``cu_seqlens_k[b]:cu_seqlens_k[b + 1]`` of ``k`` and ``v``
    (``cu_seqlens_k`` None: the same).  With ``causal``, query row ``i`` of ``Lq`` sees
    the keys ``j <= Lk - Lq + i`` (a prompt's tail over a longer prefix), else every
    key of its sequence; a row that sees none is 0.  Rows of ``out`` that belong to no
    sequence are left as they were, and rows of ``k``/``v`` that belong to none may
    hold anything; the keys and values of a sequence must be finite.

    ``max_seqlen_k`` is the longest key sequence (None: ``max_seqlen_q``, or all keys
    where ``cu_seqlens_k`` is given); it only bounds how far keys are split.  The scores, the softmax statistics and the output
    are held in fp32; the softmax weights are rounded to the element type for the
    second product.
    """
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError("expected q=[T,H,D] and k/v=[Tk,kv_heads,D]")
    q_shape, k_shape = q.shape, k.shape
    if out.shape != q_shape or k_shape != v.shape:
        raise ValueError("out must match q and k/v must have identical shapes")
    same_k = cu_seqlens_k is None
    if same_k:
        cu_seqlens_k = cu_seqlens_q
    dev = q.device
    if not (dev == k.device == v.device == out.device == cu_seqlens_q.device == cu_seqlens_k.device):
        raise ValueError("all tensors must be on the same device")
    if cu_seqlens_q.ndim != 1 or cu_seqlens_q.shape != cu_seqlens_k.shape or cu_seqlens_q.shape[0] < 1:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must contain one entry per sequence plus one")
    len_dtype = cu_seqlens_q.dtype
    if cu_seqlens_k.dtype != len_dtype or len_dtype not in _INDEX_TYPES:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must be int32 or int64 of one dtype")
    total_q, hq, head_dim = q_shape
    total_k, hkv, dk = k_shape
    if dk != head_dim or head_dim not in (64, 128, 256) or hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError("unsupported head shape for prompt attention")
    if same_k and total_k < total_q:
        raise ValueError("k and v hold fewer rows than q: pass cu_seqlens_k")
    if max_seqlen_k is None:
        max_seqlen_k = max_seqlen_q if same_k else total_k
    if not 0.0 < softmax_scale <= _lib.MAX_SOFTMAX_SCALE:
        raise ValueError("softmax_scale must be positive and at most 2e38")
    if not q.is_cuda:
        raise RuntimeError("prompt_attention runs on CUDA tensors only (no CPU path)")
    dtype = q.dtype
    if dtype not in _ELEMENT_TYPES or not (dtype == k.dtype == v.dtype == out.dtype):
        raise RuntimeError("the sm_100a kernel takes bf16 or f16 q/k/v/out of one dtype")
    (qt, qh, qd), (kt, kh, kd), (vt, vh, vd), (ot, oh, od) = q.stride(), k.stride(), v.stride(), out.stride()
    if not (qd == kd == vd == od == 1):
        raise RuntimeError("the head dimension of q, k, v and out must be contiguous")
    num_seqs = cu_seqlens_q.shape[0] - 1
    if total_q == 0 or num_seqs == 0:
        return out
    # A dimension of one element may carry any stride: it counts as packed.
    if hq == 1:
        qh = oh = head_dim
    if hkv == 1:
        kh = vh = head_dim
    if total_q == 1:
        qt, ot = hq * qh, hq * oh
    if total_k == 1:
        kt, vt = hkv * kh, hkv * vh
    if not (cu_seqlens_q.is_contiguous() and cu_seqlens_k.is_contiguous()):
        cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    max_seqlen_k = int(max_seqlen_k)
    lib = _lib.load()
    with _lib.on_device(dev):
        nbytes = _lib.varlen_workspace_bytes(dev.index, total_q, num_seqs, hq, hkv, head_dim, max_seqlen_k)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p = _lib.PromptAttnParams(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
            qt, qh, kt, kh, vt, vh, ot, oh, _lib.dtype_code(len_dtype), _lib.dtype_code(dtype), num_seqs, total_q, total_k,
            hq, hkv, head_dim, max_seqlen_k, bool(causal), softmax_scale, ws.data_ptr(), nbytes,
        )
        _lib.check(lib.b200_prompt_attn_fwd(ctypes.byref(p), _lib.current_stream(dev)), "prompt_attention")
    return out


__all__ = ["prompt_attention"]
