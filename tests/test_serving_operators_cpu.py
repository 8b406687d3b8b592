"""Refusals and host logic of prompt attention, draft-tree attention and the page operators (no GPU)."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch

import minicpm_b200
from minicpm_b200 import _lib, kv_pages, paged_tree_attention, prompt_attention
from oracle import prompt_attention_reference, tree_attention_reference
from oracle.paged_sdpa import paged_attention_reference

BF = torch.bfloat16


def _prompt(**over):
    q, k = torch.zeros(8, 4, 64, dtype=BF), torch.zeros(8, 2, 64, dtype=BF)
    args = dict(q=q, k=k, v=k.clone(), out=torch.empty_like(q), cu_seqlens_q=torch.tensor([0, 8], dtype=torch.int32),
                max_seqlen_q=8, softmax_scale=0.1)
    args.update(over)
    return args


@pytest.mark.parametrize(
    "over,error,msg",
    [
        (dict(q=torch.zeros(8, 256)), ValueError, "expected q=[T,H,D]"),
        (dict(out=torch.zeros(7, 4, 64)), ValueError, "out must match q"),
        (dict(v=torch.zeros(9, 2, 64)), ValueError, "out must match q"),
        (dict(cu_seqlens_q=torch.zeros(1, 2, dtype=torch.int32)), ValueError, "one entry per sequence plus one"),
        (dict(cu_seqlens_q=torch.zeros(0, dtype=torch.int32)), ValueError, "one entry per sequence plus one"),
        (dict(cu_seqlens_k=torch.zeros(3, dtype=torch.int32)), ValueError, "one entry per sequence plus one"),
        (dict(cu_seqlens_k=torch.zeros(2, dtype=torch.int64)), ValueError, "of one dtype"),
        (dict(cu_seqlens_q=torch.zeros(2)), ValueError, "int32 or int64"),
        (dict(k=torch.zeros(8, 3, 64), v=torch.zeros(8, 3, 64)), ValueError, "unsupported head shape"),
        (dict(k=torch.zeros(8, 2, 128), v=torch.zeros(8, 2, 128)), ValueError, "unsupported head shape"),
        (dict(q=torch.zeros(8, 4, 96), out=torch.zeros(8, 4, 96)), ValueError, "unsupported head shape"),
        (dict(k=torch.zeros(5, 2, 64), v=torch.zeros(5, 2, 64)), ValueError, "pass cu_seqlens_k"),
        (dict(softmax_scale=0.0), ValueError, "softmax_scale"),
        (dict(softmax_scale=float("nan")), ValueError, "softmax_scale"),
        (dict(softmax_scale=float("inf")), ValueError, "softmax_scale"),
        (dict(), RuntimeError, "CUDA tensors only"),
    ],
)
def test_prompt_attention_refusals(over, error, msg):
    with pytest.raises(error, match=re.escape(msg)):
        prompt_attention(**_prompt(**over))


def _tree(**over):
    q, k = torch.zeros(5, 4, 64, dtype=BF), torch.zeros(3, 16, 2, 64, dtype=BF)
    args = dict(q=q, k=k, v=k.clone(), out=torch.empty_like(q), tree_mask=torch.ones(5, 5, dtype=torch.bool),
                block_table=torch.zeros(1, 3, dtype=torch.int32), seqused_k=torch.tensor([9], dtype=torch.int32),
                cu_seqlens_q=torch.tensor([0, 5], dtype=torch.int32), max_seqlen_q=5, max_seqlen_k=9, softmax_scale=0.1)
    args.update(over)
    return args


@pytest.mark.parametrize(
    "over,error,msg",
    [
        (dict(q=torch.zeros(5, 256)), ValueError, "expected q=[T,H,D]"),
        (dict(out=torch.zeros(5, 4, 32)), ValueError, "out must match q"),
        (dict(tree_mask=torch.ones(4, 5, dtype=torch.bool)), ValueError, "one row per query token"),
        (dict(tree_mask=torch.ones(5, 5)), ValueError, "bool or uint8"),
        (dict(tree_mask=torch.ones(5, 4, dtype=torch.bool)), ValueError, "a column for each"),
        (dict(block_table=torch.zeros(1, 3)), ValueError, "integer physical block ids"),
        (dict(block_table=torch.zeros(2, 3, dtype=torch.int32)), ValueError, "same request count"),
        (dict(block_table=torch.zeros(1, 0, dtype=torch.int32)), RuntimeError, "CUDA tensors only"),
        (dict(cu_seqlens_q=torch.zeros(3, dtype=torch.int32)), ValueError, "one entry per request plus one"),
        (dict(cu_seqlens_q=torch.zeros(2, dtype=torch.int64)), ValueError, "of one dtype"),
        (dict(seqused_k=torch.zeros(1, 1, dtype=torch.int32)), ValueError, "one-dimensional"),
        (dict(k=torch.zeros(3, 8, 2, 64), v=torch.zeros(3, 8, 2, 64)), ValueError, "unsupported head shape"),
        (dict(softmax_scale=-0.1), ValueError, "softmax_scale"),
        (dict(), RuntimeError, "CUDA tensors only"),
    ],
)
def test_tree_attention_refusals(over, error, msg):
    with pytest.raises(error, match=re.escape(msg)):
        paged_tree_attention(**_tree(**over))


def _cache(**over):
    shape = dict(pool=6, page=16, heads=2, dim=64)
    shape.update(over)
    return torch.zeros(shape["pool"], 2, shape["page"], shape["heads"], shape["dim"], dtype=BF)


@pytest.mark.parametrize(
    "caches,msg",
    [
        ([], "1 to 256"),
        ([_cache()] * 2, "named twice"),
        ([_cache(), _cache(pool=7)], "must share shape"),
        ([_cache(), _cache().half()], "must share shape"),
        ([torch.zeros(6, 3, 16, 2, 64)], "a cache is"),
        ([torch.zeros(6, 16, 128)], "a cache is"),
        ([_cache()[:, :, :, :1]], "one dense run"),
        ([_cache()[..., :32]], "one dense run"),
        ([_cache(pool=0)], "must not be empty"),
        ([_cache()[..., ::2]], "rows must be contiguous"),
        ([torch.zeros(6, 2, 16, 1, 3, dtype=torch.int8)], "4-byte aligned"),
        ([_cache() for _ in range(129)], "1 to 256"),
    ],
)
def test_cache_layers_refusals(caches, msg):
    with pytest.raises(ValueError, match=re.escape(msg)):
        kv_pages.cache_layers(caches)


def test_cache_layers_layouts():
    a, b = _cache(), _cache()
    layers = kv_pages.cache_layers([a, b])
    assert layers.params.num_caches == 4 and layers.num_blocks == 6 and layers.block_size == 16
    assert kv_pages.cache_layers(layers) is layers
    assert (layers.params.row_bytes, layers.params.stride_head, layers.params.stride_tok) == (128, 128, 256)
    hnd = torch.zeros(6, 2, 2, 16, 64, dtype=BF).permute(0, 1, 3, 2, 4)
    p = kv_pages.cache_layers([hnd]).params
    assert (p.stride_tok, p.stride_head, p.stride_block) == (128, 16 * 128, 4 * 16 * 128)
    p = kv_pages.cache_layers([_cache(pool=1, heads=1)]).params
    assert (p.stride_head, p.stride_tok, p.stride_block) == (128, 128, 16 * 128)


def _pool(**over):
    args = dict(kv_caches=[_cache()], block_table=torch.full((3, 4), -1, dtype=torch.int32),
                seq_lens=torch.zeros(3, dtype=torch.int32), ref_counts=torch.zeros(6, dtype=torch.int32),
                parents=torch.tensor([0]), children=torch.tensor([1]))
    args.update(over)
    return args


@pytest.mark.parametrize(
    "over,error,msg",
    [
        (dict(parents=torch.tensor([0.0])), ValueError, "parents must be"),
        (dict(children=torch.tensor([1, 2])), ValueError, "one length and dtype"),
        (dict(children=torch.tensor([1], dtype=torch.int32)), ValueError, "one length and dtype"),
        (dict(block_table=torch.zeros(3, 4)), ValueError, "integer physical block ids"),
        (dict(block_table=torch.zeros(4, 3, dtype=torch.int32).t()), ValueError, "written in place"),
        (dict(block_table=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)), ValueError, "written in place"),
        (dict(seq_lens=torch.zeros(4, dtype=torch.int32)), ValueError, "one int32 or int64 length"),
        (dict(seq_lens=torch.zeros(6, dtype=torch.int32)[::2]), ValueError, "contiguous"),
        (dict(ref_counts=torch.zeros(5, dtype=torch.int32)), ValueError, "one int32 per page"),
        (dict(ref_counts=torch.zeros(6, dtype=torch.int64)), ValueError, "one int32 per page"),
        (dict(ref_counts=None), ValueError, "needs ref_counts"),
        (dict(), RuntimeError, "CUDA tensors only"),
    ],
)
def test_fork_refusals(over, error, msg):
    with pytest.raises(error, match=re.escape(msg)):
        kv_pages.fork_sequences(**_pool(**over))


def test_copy_free_and_keep_refusals():
    with pytest.raises(ValueError, match="one length"):
        kv_pages.copy_pages([_cache()], torch.tensor([1, 2]), torch.tensor([3]))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kv_pages.copy_pages([_cache()], torch.tensor([1]), torch.tensor([3]))
    p = _pool()
    state = (p["block_table"], p["seq_lens"], p["ref_counts"])
    with pytest.raises(ValueError, match="rows must be"):
        kv_pages.free_sequences(*state, torch.tensor([[0]]))
    with pytest.raises(ValueError, match="needs ref_counts"):
        kv_pages.free_sequences(state[0], state[1], None, torch.tensor([0]))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        kv_pages.free_sequences(*state, torch.tensor([0]))
    acc, num, ctx = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)

    def keep(table=state[0], context=ctx, accepted=acc, counts=num, lens=state[1]):
        kv_pages.keep_accepted_tokens(p["kv_caches"], table, context, accepted, counts, lens)

    for over, msg in [(dict(context=ctx.long()), "must match seq_lens"), (dict(accepted=acc[:2]), "one row per row"),
                      (dict(counts=num.long()), "dtype of accepted"), (dict(counts=num[:2]), "one count per row"),
                      (dict(lens=ctx), "context_lens"),
                      (dict(context=torch.zeros(9, dtype=torch.int32)[1:4], lens=None), "context_lens")]:
        if over.get("lens", 0) is None:  # two views of one buffer that overlap
            over["lens"] = over["context"].as_strided((3,), (1,), 0)
        with pytest.raises(ValueError, match=msg):
            keep(**over)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        keep()


@pytest.mark.parametrize("lens_type", [torch.int32, torch.int64])
def test_keep_refuses_counts_that_its_lengths_overwrite(lens_type):
    # Several warps read a sequence's count; the first to finish stores its length.
    p = _pool(seq_lens=torch.zeros(3, dtype=lens_type))
    ctx, acc = torch.zeros(3, dtype=lens_type), torch.zeros(3, 2, dtype=torch.int32)
    shared = torch.zeros(12, dtype=torch.int32)
    for counts, at in [(shared[:3], 0), (shared[1:4], 0), (shared[2:5], 0)]:
        lens = shared.view(lens_type).as_strided((3,), (1,), at)
        with pytest.raises(ValueError, match="num_accepted"):
            kv_pages.keep_accepted_tokens(p["kv_caches"], p["block_table"], ctx, acc, counts, lens)
    lens = shared.view(lens_type)[:3]
    apart = shared[lens.element_size() // 4 * 3:][:3]
    with pytest.raises(RuntimeError, match="CUDA tensors only"):  # behind them: accepted, up to the device
        kv_pages.keep_accepted_tokens(p["kv_caches"], p["block_table"], ctx, acc, apart, lens)


def test_c_entries_return_a_status():
    lib = _lib.load()
    assert lib.b200_prompt_attn_fwd(None, None) == _lib.B200_ERR_INVALID
    assert lib.b200_tree_attn_fwd(None, None) == _lib.B200_ERR_INVALID
    p = _lib.PromptAttnParams(dtype=_lib.DTYPE_F32, num_q_heads=4, num_kv_heads=2, head_dim=64)
    assert lib.b200_prompt_attn_fwd(ctypes.byref(p), None) == _lib.B200_ERR_UNSUPPORTED
    p = _lib.PromptAttnParams(dtype=_lib.DTYPE_BF16, num_q_heads=4, num_kv_heads=2, head_dim=64, seqlen_dtype=_lib.DTYPE_I32)
    assert lib.b200_prompt_attn_fwd(ctypes.byref(p), None) == _lib.B200_ERR_INVALID
    assert "softmax_scale" in lib.b200_last_error().decode()
    p.softmax_scale = 0.5
    assert lib.b200_prompt_attn_fwd(ctypes.byref(p), None) == _lib.B200_OK  # no tokens
    p.num_q_heads, p.num_kv_heads = 129, 1
    assert lib.b200_prompt_attn_fwd(ctypes.byref(p), None) == _lib.B200_ERR_UNSUPPORTED
    t = _lib.TreeAttnParams(dtype=_lib.DTYPE_BF16, num_q_heads=4, num_kv_heads=2, head_dim=64, seqlen_dtype=_lib.DTYPE_I32,
                            softmax_scale=1.0, block_size=24)
    assert lib.b200_tree_attn_fwd(ctypes.byref(t), None) == _lib.B200_ERR_INVALID
    assert lib.b200_varlen_attn_workspace_bytes(0, 1, 4, 2, 64, 10) == 0
    assert lib.b200_varlen_attn_workspace_bytes(10, 1, 4, 0, 64, 10) == 0
    # The split bound is a bound on memory: one long sequence at 2 KV heads stays below 64 MB.
    assert 0 < lib.b200_varlen_attn_workspace_bytes(16, 1, 16, 2, 128, 1 << 20) < 1 << 26
    layers = kv_pages.cache_layers([_cache()])
    seqs = _lib.SeqTable()
    assert lib.b200_copy_pages(None, None, None, 1, _lib.DTYPE_I32, None) == _lib.B200_ERR_INVALID
    assert lib.b200_copy_pages(layers._ref, None, None, 1, _lib.DTYPE_BF16, None) == _lib.B200_ERR_INVALID
    assert lib.b200_copy_pages(layers._ref, None, None, 1, _lib.DTYPE_I32, None) == _lib.B200_ERR_INVALID
    assert lib.b200_copy_pages(layers._ref, None, None, 0, _lib.DTYPE_I32, None) == _lib.B200_OK
    assert lib.b200_fork_sequences(layers._ref, ctypes.byref(seqs), None, None, 1, 3, None, 0, None) == _lib.B200_ERR_INVALID
    assert lib.b200_free_sequences(ctypes.byref(seqs), None, 1, 3, None) == _lib.B200_ERR_INVALID
    assert lib.b200_keep_accepted(layers._ref, ctypes.byref(seqs), None, None, 0, 0, None, 3, None) == _lib.B200_ERR_INVALID
    assert lib.b200_fork_workspace_bytes(5, 7) >= 5 * 16 + 7 * 4 + 5 * 4


def test_public_names():
    for name in ("prompt_attention", "paged_tree_attention", "kv_pages"):
        assert name in minicpm_b200.__all__ and hasattr(minicpm_b200, name)


def test_the_oracles_agree_with_the_paged_one():
    """A chain draft over a permuted cache, and the same rows without a cache, in three restatements."""
    g = torch.Generator().manual_seed(1)
    q = torch.randn(7, 4, 64, generator=g)
    cache = torch.randn(4, 2, 16, 2, 64, generator=g)
    table, L = torch.tensor([[2, 0, 3]]), 39
    want = paged_attention_reference(q, cache[:, 0], cache[:, 1], table, torch.tensor([0, 7]), torch.tensor([L]), 0.3)
    mask = torch.tril(torch.ones(7, 7, dtype=torch.bool))
    tree, a, s = tree_attention_reference(q, cache[:, 0], cache[:, 1], mask, table, [L], [0, 7], 0.3)
    assert (tree - want.double()).abs().max() < 1e-5 and (a >= tree.abs() - 1e-12).all() and (s > 0).all()
    rows = cache[table[0]].transpose(0, 1).reshape(2, -1, 2, 64)[:, :L]
    plain, _, _ = prompt_attention_reference(q, rows[0], rows[1], [0, 7], [0, L], 0.3, True)
    assert (plain - tree).abs().max() < 1e-12


# ------------------------------------------------------------------ routes
def _flags(monkeypatch, on=True):
    for name in ("ILUVATAR_USE_OPTIMIZED", "ILUVATAR_SPLIT_KV"):
        if on:
            monkeypatch.setenv(name, "1")
        else:
            monkeypatch.delenv(name, raising=False)
    monkeypatch.delenv("ILUVATAR_SPLIT_KV_DECODE", raising=False)


@pytest.mark.parametrize("max_q", [1, 9])
def test_dispatcher_sends_trees_to_the_optimized_path(monkeypatch, max_q):
    from minicpm_b200 import attention

    seen = {}
    monkeypatch.setattr(attention, "unified_attention_optimized", lambda **kw: seen.update(kw))
    monkeypatch.setattr(attention, "_vllm_unified_attention", lambda: pytest.fail("a tree has no baseline"))
    q, k = torch.zeros(9, 16, 128, dtype=BF), torch.zeros(4, 16, 2, 128, dtype=BF)
    mask = torch.ones(9, 9, dtype=torch.bool)
    args = (q, k, k, q, None, max_q, None, 64, 0.1)
    _flags(monkeypatch, False)
    with pytest.raises(RuntimeError, match="optimized path only"):
        minicpm_b200.iluvatar_attention(*args, tree_mask=mask)
    _flags(monkeypatch)
    minicpm_b200.iluvatar_attention(*args, tree_mask=mask)
    assert seen["tree_mask"] is mask and seen["max_seqlen_q"] == max_q
    with pytest.raises(RuntimeError, match="optimized path only"):
        minicpm_b200.iluvatar_attention(*args, tree_mask=mask, softcap=30.0)


def test_service_routes_trees_and_encoders(monkeypatch):
    from types import SimpleNamespace

    from minicpm_b200 import service

    calls = []
    monkeypatch.setattr(service, "unified_attention_optimized", lambda **kw: calls.append(("tree", kw)))
    monkeypatch.setattr(service, "_vllm_unified_attention", lambda: (lambda **kw: calls.append(("vllm", kw))))
    monkeypatch.setattr(service, "prompt_attention", lambda *a, **kw: calls.append(("prompt", a, kw)))
    q, k = torch.zeros(9, 16, 128, dtype=BF), torch.zeros(4, 16, 2, 128, dtype=BF)
    mask = torch.ones(9, 9, dtype=torch.bool)
    base = dict(q=q, k=k, v=k, out=q, cu_seqlens_q=None, max_seqlen_q=1, seqused_k=None, max_seqlen_k=64, softmax_scale=0.1,
                causal=True, block_table=None)
    _flags(monkeypatch, False)
    with pytest.raises(RuntimeError, match="sm_100a path only"):
        service._run_unified_attention(**base, tree_mask=mask)
    service._run_unified_attention(**base, tree_mask=None)
    assert calls[-1][0] == "vllm" and "tree_mask" not in calls[-1][1]
    _flags(monkeypatch)
    service._run_unified_attention(**base, tree_mask=mask)
    assert calls[-1][0] == "tree" and calls[-1][1]["tree_mask"] is mask
    with pytest.raises(RuntimeError, match="sm_100a path only"):
        service._run_unified_attention(**{**base, "causal": False}, tree_mask=mask)

    # The metadata carries the mask of the step; a scheduler without one leaves it out.
    common = SimpleNamespace(num_reqs=1, num_actual_tokens=9, max_query_len=9, max_seq_len=64,
                             query_start_loc=torch.tensor([0, 9]), seq_lens=torch.tensor([64]),
                             block_table_tensor=torch.zeros(1, 4), slot_mapping=None, causal=True)
    builder = service.IluvatarAttentionMetadataBuilder(16, 2, 128, torch.device("cpu"))
    assert builder.build(0, common).tree_mask is None
    common.tree_mask = torch.ones(12, 9, dtype=torch.bool)  # padded like the step's tensors
    meta = builder.build(0, common)
    impl = service.IluvatarAttentionImpl(16, 128, 0.1, 2, None, None, "auto")
    impl.forward(SimpleNamespace(), q, q, q, torch.zeros(4, 2, 16, 2, 128, dtype=BF), meta, torch.empty_like(q))
    assert calls[-1][0] == "tree" and calls[-1][1]["tree_mask"].shape == (9, 9)

    # Encoder batches: the sm_100a kernel with both flags and a plain call, else vLLM's.
    meta.tree_mask = None
    enc = service.IluvatarAttentionImpl(16, 128, 0.1, 2, None, None, "auto", attn_type=service.AttentionType.ENCODER_ONLY)
    kv = torch.zeros(9, 2, 128, dtype=BF)
    enc.forward(SimpleNamespace(), q, kv, kv, torch.zeros(0), meta, torch.empty_like(q))
    assert calls[-1][0] == "prompt" and calls[-1][2] == {"causal": False}
    count = len(calls)
    for over in (dict(sliding_window=128), dict(alibi_slopes=[0.1] * 16), dict(logits_soft_cap=30.0)):
        args = dict(alibi_slopes=None, sliding_window=None, logits_soft_cap=None)
        args.update(over)
        other = service.IluvatarAttentionImpl(16, 128, 0.1, 2, args["alibi_slopes"], args["sliding_window"], "auto",
                                              args["logits_soft_cap"], attn_type=service.AttentionType.ENCODER_ONLY)
        try:
            other.forward(SimpleNamespace(), q, kv, kv, torch.zeros(0), meta, torch.empty_like(q))
        except Exception:
            pass  # vLLM's kernel does not run here
        assert len(calls) == count
