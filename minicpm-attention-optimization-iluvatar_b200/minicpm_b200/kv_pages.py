"""Page operators of a paged KV cache on sm_100a: copy, fork, free, keep.

For serving that branches: parallel samples and beams share their prompt's pages
(:func:`fork_sequences`, :func:`free_sequences`), a scheduler duplicates pages before
they are written to (:func:`copy_pages`), and speculative decoding keeps the accepted
path of a draft (:func:`keep_accepted_tokens`).  Every call serves all layers in one
launch, on the current CUDA stream, without a host synchronisation, and can be
captured in a CUDA graph.  No counterpart in the reference.

A pool's state is three tensors that the caller owns: ``block_table [max_seqs,
max_pages]`` (-1 = no page), ``seq_lens [max_seqs]`` and ``ref_counts [num_blocks]``
(int32, how many rows of the table name a page; 0 = free).  What a call cannot serve
(an index out of range, no page left) is skipped, leaves the other entries alone, and
is recorded in the device error word (``minicpm_b200._lib.device_error()``).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import torch

from . import _lib


class CacheLayers:
    """The K and V tensors of a model's layers, checked once (:func:`cache_layers`).

    Holds the tensors, so their memory stays valid; what is written to them later is
    seen by every call.
    """

    def __init__(self, kv_caches: Sequence[torch.Tensor]):
        caches = list(kv_caches)
        if not caches:
            raise ValueError("1 to 256 K/V tensors (128 layers) in one set of caches")
        first = caches[0]
        shape, strides, dtype, device = first.shape, first.stride(), first.dtype, first.device
        paired = len(shape) == 5 and shape[1] == 2
        if not paired and len(shape) != 4:
            raise ValueError("a cache is [num_blocks, 2, block_size, kv_heads, D] or [num_blocks, block_size, kv_heads, D]")
        e = first.element_size()
        base: list[int] = []
        for t in caches:
            if t.shape != shape or t.stride() != strides or t.dtype != dtype or t.device != device:
                raise ValueError("all caches must share shape, strides, dtype and device")
            base.append(t.data_ptr())
            if paired:
                base.append(base[-1] + strides[1] * e)
        if len(base) > 256:
            raise ValueError("1 to 256 K/V tensors (128 layers) in one set of caches")
        n, block, heads, row = (shape[0], *shape[2:]) if paired else shape
        sb, st, sh, sd = (strides[0], *strides[2:]) if paired else strides
        if n * block * heads * row == 0 or (sd != 1 and row != 1):
            raise ValueError("the caches must not be empty and their rows must be contiguous")
        if len(set(base)) != len(base):
            raise ValueError("a cache is named twice")
        page = block * heads * row
        nhd = (heads == 1 or sh == row) and (block == 1 or st == heads * row)
        hnd = (block == 1 or st == row) and (heads == 1 or sh == block * row)
        if not (nhd or hnd) or (n > 1 and sb < page):
            raise ValueError("a page must be one dense run of [block_size, kv_heads, D] or [kv_heads, block_size, D]")
        # A dimension of one element may carry any stride: the library gets the dense one.
        if n == 1:
            sb = page
        if block == 1:
            st = heads * row if nhd else row
        if heads == 1:
            sh = row
        if (sb * e) % 4 or (row * e) % 4 or any(b % 4 for b in base):
            raise ValueError("cache rows must be 4-byte aligned")
        self.tensors = caches
        self.device = device
        self.num_blocks, self.block_size = n, block
        self._base = (ctypes.c_void_p * len(base))(*base)
        self.params = _lib.PageCaches(ctypes.cast(self._base, ctypes.c_void_p), len(base), n, block, heads, row * e, sb * e,
                                      st * e, sh * e)
        self._ref = ctypes.byref(self.params)


Caches = Union[CacheLayers, Sequence[torch.Tensor]]


def cache_layers(kv_caches: Caches) -> CacheLayers:
    """Check a model's caches once and keep them together for the calls below.

    ``kv_caches``: one ``[num_blocks, 2, block_size, kv_heads, D]`` tensor per layer, or K and
    V tensors ``[num_blocks, block_size, kv_heads, D]``; of one shape, one layout (NHD, or a
    permuted view of HND) and any element type, quantised ones included (rows are moved with
    the scale that they carry inline).
    """
    return kv_caches if isinstance(kv_caches, CacheLayers) else CacheLayers(kv_caches)


_INDEX_CODES = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}


def _indices(name: str, t: torch.Tensor, device: torch.device) -> tuple[torch.Tensor, int, int]:
    """``t`` (contiguous), its length and the code of its dtype."""
    code = _INDEX_CODES.get(t.dtype)
    if code is None or t.ndim != 1:
        raise ValueError(f"{name} must be a one-dimensional int32 or int64 tensor")
    if t.device != device:
        raise ValueError(f"{name} must be on the same device as the table or caches")
    return t if t.is_contiguous() else t.contiguous(), t.shape[0], code


def _table(block_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: Optional[torch.Tensor], num_blocks: int,
           block_size: int) -> tuple["_lib.SeqTable", int, torch.device]:
    """The table as the library takes it, its rows and its device."""
    code, len_code = _INDEX_CODES.get(block_table.dtype), _INDEX_CODES.get(seq_lens.dtype)
    if code is None or block_table.ndim != 2:
        raise ValueError("block_table must contain integer physical block ids, [max_seqs, max_pages]")
    rows, cols = block_table.shape
    if cols == 0:
        raise ValueError("block_table must contain integer physical block ids, [max_seqs, max_pages]")
    stride, step = block_table.stride()
    if step != 1 or (rows > 1 and stride < cols):
        raise ValueError("block_table is written in place: its rows must be contiguous and apart")
    if len_code is None or seq_lens.ndim != 1 or seq_lens.shape[0] != rows:
        raise ValueError("seq_lens must hold one int32 or int64 length per row of the block table")
    if not seq_lens.is_contiguous():
        raise ValueError("seq_lens is written in place: it must be contiguous")
    dev = block_table.device
    if seq_lens.device != dev:
        raise ValueError("block_table and seq_lens must be on the same device")
    refs = None
    if ref_counts is not None:
        if ref_counts.ndim != 1 or ref_counts.dtype is not torch.int32 or ref_counts.shape[0] != num_blocks:
            raise ValueError("ref_counts must hold one int32 per page")
        if not ref_counts.is_contiguous() or ref_counts.device != dev:
            raise ValueError("ref_counts is written in place: contiguous, on the table's device")
        refs = ref_counts.data_ptr()
    table = _lib.SeqTable(block_table.data_ptr(), seq_lens.data_ptr(), refs, stride if rows > 1 else max(stride, cols), cols,
                          rows, num_blocks, block_size, code, len_code)
    return table, rows, dev


def _on(layers: CacheLayers, dev: torch.device, what: str) -> None:
    if layers.device != dev:
        raise ValueError("the caches and the indices must be on the same device")
    if dev.type != "cuda":
        raise RuntimeError(f"{what} runs on CUDA tensors only (no CPU path)")


def copy_pages(kv_caches: Caches, src_pages: torch.Tensor, dst_pages: torch.Tensor) -> None:
    """Copy page ``src_pages[i]`` to page ``dst_pages[i]`` in every layer's K and V.

    A pair with a negative index is padding.  A destination may be neither named twice nor
    a source of another pair: the copies run at the same time.
    """
    layers = cache_layers(kv_caches)
    dev = layers.device
    src, n, code = _indices("src_pages", src_pages, dev)
    dst, n_dst, dst_code = _indices("dst_pages", dst_pages, dev)
    if n != n_dst or code != dst_code:
        raise ValueError("src_pages and dst_pages must have one length and dtype")
    _on(layers, dev, "copy_pages")
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.b200_copy_pages(layers._ref, src.data_ptr(), dst.data_ptr(), n, code, _lib.current_stream(dev)),
                   "copy_pages")


def fork_sequences(kv_caches: Caches, block_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor,
                   parents: torch.Tensor, children: torch.Tensor) -> None:
    """Make row ``children[i]`` of the table a copy of row ``parents[i]``, for every ``i``.

    Full pages are shared and their counts rise; the used rows of a partial last page are
    copied, in every layer, to a page of the child's own: the lowest free pages, given out in
    the order of the entries.  The child's row must have length 0 and is named once; pages that
    it names all the same (reserved ones) are released, and are not given out by the same call.  A
    parent may have any number of children.  Entries with a negative index are padding; one
    that cannot be served leaves its child as it was and is recorded.  A full page that the
    parent's row does not name is missing in the child's row too (-1), and is recorded.
    """
    layers = cache_layers(kv_caches)
    table, rows, dev = _table(block_table, seq_lens, ref_counts, layers.num_blocks, layers.block_size)
    if ref_counts is None:
        raise ValueError("fork_sequences needs ref_counts")
    p, n, code = _indices("parents", parents, dev)
    c, n_children, c_code = _indices("children", children, dev)
    if n != n_children or code != c_code:
        raise ValueError("parents and children must have one length and dtype")
    _on(layers, dev, "fork_sequences")
    if n == 0:
        return
    lib = _lib.load()
    with _lib.on_device(dev):
        nbytes = _lib.fork_workspace_bytes(n, rows)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.check(lib.b200_fork_sequences(layers._ref, ctypes.byref(table), p.data_ptr(), c.data_ptr(), n, code,
                                           ws.data_ptr(), nbytes, _lib.current_stream(dev)), "fork_sequences")


def free_sequences(block_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor,
                   rows: torch.Tensor) -> None:
    """Empty the rows named: their pages' counts fall, their entries become -1, their lengths 0.

    A page whose count reaches 0 is free.  Naming a row twice, or an empty one, releases
    nothing twice; negative rows are padding.
    """
    if ref_counts is None:
        raise ValueError("free_sequences needs ref_counts")
    table, _, dev = _table(block_table, seq_lens, ref_counts, max(ref_counts.numel(), 1), 1)
    r, n, code = _indices("rows", rows, dev)
    if dev.type != "cuda":
        raise RuntimeError("free_sequences runs on CUDA tensors only (no CPU path)")
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.b200_free_sequences(ctypes.byref(table), r.data_ptr(), n, code, _lib.current_stream(dev)),
                   "free_sequences")


def keep_accepted_tokens(kv_caches: Caches, block_table: torch.Tensor, context_lens: torch.Tensor,
                         accepted: torch.Tensor, num_accepted: torch.Tensor, seq_lens: torch.Tensor,
                         ref_counts: Optional[torch.Tensor] = None) -> None:
    """Move the accepted drafted tokens of every sequence together, behind its context.

    For row ``b`` and ``i < num_accepted[b]``, the K/V row at position ``context_lens[b] +
    accepted[b, i]`` goes to ``context_lens[b] + i`` in every layer, and ``seq_lens[b]`` becomes
    ``context_lens[b] + num_accepted[b]``.  ``accepted`` ``[num_seqs, A]`` holds the path's indices
    among the drafted tokens, strictly rising; what is behind ``num_accepted[b]`` is not read.
    With ``ref_counts`` the pages behind the new lengths are released (their table entries
    become -1) and a shared page is not written to.  ``seq_lens`` may overlap neither
    ``context_lens`` nor ``num_accepted``.  A path is cut before its first entry
    that does not rise or has no page of its own, which is recorded; a negative context is
    recorded too, its row keeps its pages and gets length 0.
    """
    layers = cache_layers(kv_caches)
    table, rows, dev = _table(block_table, seq_lens, ref_counts, layers.num_blocks, layers.block_size)
    if context_lens.shape != seq_lens.shape or context_lens.dtype != seq_lens.dtype or context_lens.device != dev:
        raise ValueError("context_lens must match seq_lens")
    if accepted.ndim != 2 or accepted.shape[0] != rows or accepted.device != dev:
        raise ValueError("accepted must have one row per row of the block table")
    counts, n, code = _indices("num_accepted", num_accepted, dev)
    if n != rows or counts.dtype != accepted.dtype:
        raise ValueError("num_accepted must hold one count per row, in the dtype of accepted")
    # Other sequences' lengths, counts and paths are read while seq_lens is written.
    lens_begin, lens_bytes = seq_lens.data_ptr(), rows * seq_lens.element_size()
    index_bytes, counts_begin = counts.element_size(), counts.data_ptr()
    if abs(context_lens.data_ptr() - lens_begin) < lens_bytes:
        raise ValueError("seq_lens may not be (or overlap) context_lens")
    if counts_begin < lens_begin + lens_bytes and lens_begin < counts_begin + rows * index_bytes:
        raise ValueError("seq_lens may not be (or overlap) num_accepted")
    _on(layers, dev, "keep_accepted_tokens")
    most = accepted.shape[1]
    stride, step = accepted.stride()
    if most and (step != 1 or stride < most):
        accepted = accepted.contiguous()
        stride = most
    accepted_begin = accepted.data_ptr()
    if accepted_begin < lens_begin + lens_bytes and lens_begin < accepted_begin + rows * stride * index_bytes:
        accepted = accepted.clone(memory_format=torch.contiguous_format)
        accepted_begin, stride = accepted.data_ptr(), most
    context_lens = context_lens.contiguous()
    lib = _lib.load()
    with _lib.on_device(dev):
        _lib.check(lib.b200_keep_accepted(layers._ref, ctypes.byref(table), context_lens.data_ptr(), accepted_begin,
                                          max(stride, most), most, counts_begin, code, _lib.current_stream(dev)),
                   "keep_accepted_tokens")


__all__ = [
    "CacheLayers",
    "cache_layers",
    "copy_pages",
    "fork_sequences",
    "free_sequences",
    "keep_accepted_tokens",
]
