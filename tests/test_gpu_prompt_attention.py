"""Packed prompt attention against its 64-bit definition (GPU): types, head shapes, lengths
from one token on, causal and bidirectional, longer keys than queries, strides, garbage
around the sequences, streams, graphs and concurrent calls."""

from __future__ import annotations

import threading

import pytest
import torch

from minicpm_b200 import _lib, paged_split_kv_attention, prompt_attention
from oracle import attention_tolerance, prompt_attention_reference

pytestmark = pytest.mark.gpu


def _cu(lens, dtype=torch.int32):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=dtype)


def _inputs(ql, kl, hq, hkv, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(ql), hq, dim, generator=g).to(dtype)
    k = torch.randn(sum(kl), hkv, dim, generator=g).to(dtype)
    v = torch.randn(sum(kl), hkv, dim, generator=g).to(dtype)
    return q, k, v


def _check(out, q, k, v, ql, kl, scale, causal, tag=""):
    o, a, s = prompt_attention_reference(q, k, v, _cu(ql).tolist(), _cu(kl).tolist(), scale, causal)
    tol = attention_tolerance(o, a, s, max(kl), q.shape[2], q.dtype, v.double().abs().max().item())
    d = (out.cpu().double() - o).abs()
    assert torch.isfinite(d).all(), f"{tag}: non-finite output"
    worst = (d / tol).max().item()
    assert worst <= 1.0, f"{tag}: {worst:.2f} of the bound"
    assert _lib.device_error() == _lib.DEVERR_NONE


def _run(ql, kl, hq, hkv, dim, dtype, causal, seed=0):
    q, k, v = _inputs(ql, kl, hq, hkv, dim, dtype, seed)
    out = torch.full(q.shape, float("nan"), dtype=dtype, device="cuda")
    scale = dim ** -0.5
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), out, _cu(ql).cuda(), max(ql), scale, causal=causal,
                           cu_seqlens_k=_cu(kl).cuda(), max_seqlen_k=max(kl))
    assert got is out
    torch.cuda.synchronize()
    _check(out, q, k, v, ql, kl, scale, causal, f"{ql} {kl} {hq}/{hkv}x{dim} {dtype} causal={causal}")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_types_and_head_dims(dim, dtype, causal):
    _run([1, 17, 130, 255, 64], [1, 17, 130, 255, 64], 8, 2, dim, dtype, causal, seed=dim)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv", [(16, 2), (12, 12), (1, 1), (6, 1), (24, 8), (128, 1), (20, 10)])
def test_head_groups(hq, hkv, causal):
    _run([5, 70, 129], [5, 70, 129], hq, hkv, 64, torch.bfloat16, causal, seed=hq)


@pytest.mark.parametrize("n", [1, 2, 127, 128, 129, 255, 256, 257, 511, 1000])
def test_lengths_around_the_tiles(n):
    _run([n], [n], 4, 2, 64, torch.bfloat16, True, seed=n)
    _run([n, n], [n, n], 2, 2, 64, torch.float16, False, seed=n)


def test_one_long_sequence_is_split_over_the_keys():
    # Few units for 148 SMs: the keys are split and combined.
    _run([40], [5000], 8, 2, 128, torch.bfloat16, True)
    _run([3], [9001], 8, 1, 64, torch.float16, False)
    _run([33], [3001], 4, 1, 256, torch.bfloat16, True)


@pytest.mark.parametrize("causal", [True, False])
def test_longer_and_shorter_keys_and_empty_sequences(causal):
    # Keys longer than the queries, shorter (rows without a key are 0), no query, no key.
    ql, kl = [7, 50, 0, 20, 4, 1], [300, 50, 10, 12, 0, 2]
    q, k, v = _inputs(ql, kl, 8, 2, 128, torch.bfloat16, 5)
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    prompt_attention(q.cuda(), k.cuda(), v.cuda(), out, _cu(ql).cuda(), 50, 0.1, causal=causal, cu_seqlens_k=_cu(kl).cuda(),
                     max_seqlen_k=300)
    _check(out, q, k, v, ql, kl, 0.1, causal)
    if causal:
        assert out[57:65].abs().max().item() == 0.0
    assert out[77:81].abs().max().item() == 0.0


def test_no_keys_at_all():
    q = torch.randn(5, 4, 64, device="cuda", dtype=torch.bfloat16)
    kv = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 3.0)
    zero = torch.zeros(2, device="cuda", dtype=torch.int32)
    prompt_attention(q, kv, kv, out, torch.tensor([0, 5], device="cuda", dtype=torch.int32), 5, 0.1, cu_seqlens_k=zero,
                     max_seqlen_k=0)
    assert out.abs().max().item() == 0.0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_garbage_around_the_sequences(dim, causal):
    """NaN rows before, between and behind the sequences of k / v; rows of out behind them stay."""
    ql = [70, 131, 9]
    q, k, v = _inputs(ql, ql, 8, 2, dim, torch.bfloat16, 3)
    gap = 5
    rows, big = [], []
    kb = torch.full((sum(ql) + 4 * gap, 2, dim), float("nan"), dtype=q.dtype)
    vb = torch.full_like(kb, float("inf"))
    cu, at, src = [], gap, 0
    # Sequences with a gap between them: one call per sequence's neighbours is not needed, the
    # gaps become sequences of no query rows.
    cu_q, cu_k = [0], [0]
    for n in ql:
        cu_q += [cu_q[-1], cu_q[-1] + n]
        cu_k += [cu_k[-1] + gap, cu_k[-1] + gap + n]
        kb[cu_k[-2]:cu_k[-1]], vb[cu_k[-2]:cu_k[-1]] = k[src:src + n], v[src:src + n]
        src += n
    qb = torch.randn(sum(ql) + 11, 8, dim).to(q.dtype)
    qb[:sum(ql)] = q
    out = torch.full(qb.shape, 7.0, dtype=q.dtype, device="cuda")
    prompt_attention(qb.cuda(), kb.cuda(), vb.cuda(), out, torch.tensor(cu_q, dtype=torch.int32).cuda(), 131, dim ** -0.5,
                     causal=causal, cu_seqlens_k=torch.tensor(cu_k, dtype=torch.int32).cuda(), max_seqlen_k=131)
    _check(out[:sum(ql)], q, k, v, ql, ql, dim ** -0.5, causal)
    assert (out[sum(ql):] == 7.0).all()


def test_strided_views_and_int64_lengths():
    ql = [33, 90]
    q, k, v = _inputs(ql, ql, 8, 2, 128, torch.bfloat16, 8)
    qkv = torch.zeros(sum(ql), 12, 128, dtype=torch.bfloat16)
    qkv[:, :8], qkv[:, 8:10], qkv[:, 10:] = q, k, v
    qkv = qkv.cuda()
    out = torch.zeros(sum(ql), 2, 8, 128, dtype=torch.bfloat16, device="cuda")
    cu = torch.stack([_cu(ql, torch.int64)] * 2, dim=1).cuda()[:, 0]  # not contiguous
    prompt_attention(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], out[:, 1], cu, 90, 0.09)
    _check(out[:, 1], q, k, v, ql, ql, 0.09, True)
    assert out[:, 0].abs().max().item() == 0.0
    # One row with an odd leading stride: a dimension of one element takes any stride.
    one = torch.randn(4, 7 + 8 * 128, device="cuda").to(torch.bfloat16)[1:2, 7:]
    row = torch.as_strided(torch.randn(8 * 128 + 8, device="cuda").to(torch.bfloat16), (1, 8, 128), (3, 128, 1))
    kv = k[:1].cuda()
    out1 = torch.empty_like(row)
    prompt_attention(row, kv, v[:1].cuda(), out1, torch.tensor([0, 1], device="cuda"), 1, 0.09)
    assert torch.equal(out1.view(2, 4, 128)[0, 0].cpu(), v[0, 0])
    assert one.shape[0] == 1


def test_large_scores_do_not_overflow():
    ql = [200]
    q, k, v = _inputs(ql, ql, 4, 2, 64, torch.float16, 4)
    q, k = q * 30, k * 30
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    prompt_attention(q.cuda(), k.cuda(), v.cuda(), out, _cu(ql).cuda(), 200, 0.125)
    _check(out, q, k, v, ql, ql, 0.125, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_batches_that_fill_the_gpu(dim, dtype, causal):
    """More whole units than SMs: the schedule kernel's list."""
    ql = [(37 * i) % 300 for i in range(24)]
    _run(ql, ql, 16, 8, dim, dtype, causal, seed=dim)


def test_few_rounds_of_long_units_are_shared():
    """150 equal units on 148 SMs: streamed although there are more units than SMs."""
    ql, kl = [9] * 75, [4100] * 75
    _run(ql, kl, 4, 2, 64, torch.bfloat16, True, seed=1)


@pytest.mark.parametrize("n", [64, 65, 150])
@pytest.mark.parametrize("causal", [True, False])
def test_many_short_sequences(n, causal):
    """Up to 64 sequences one warp divides the work, above that the block; one KV head keeps the batch small."""
    ql = [(7 * i) % 11 for i in range(n)]
    _run(ql, ql, 2, 1, 64, torch.bfloat16, causal, seed=n)


@pytest.mark.parametrize("hint", [0, 1, 700, 1 << 20])
def test_a_wrong_bound_of_the_longest_sequence_costs_time_only(hint):
    ql, kl = [5, 40, 0, 9], [1500, 40, 3, 700]
    q, k, v = _inputs(ql, kl, 4, 1, 128, torch.bfloat16, 2)
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    prompt_attention(q.cuda(), k.cuda(), v.cuda(), out, _cu(ql).cuda(), 40, 0.1, cu_seqlens_k=_cu(kl).cuda(), max_seqlen_k=hint)
    _check(out, q, k, v, ql, kl, 0.1, True)


def test_lengths_past_the_tensors_stay_in_bounds():
    """cu_seqlens that name rows the tensors do not have are clipped; rows behind stay as they were."""
    q, k, v = (t.cuda() for t in _inputs([64], [64], 4, 2, 64, torch.bfloat16, 6))
    want = torch.empty_like(q)
    prompt_attention(q, k, v, want, _cu([64]).cuda(), 64, 0.1)
    out = torch.empty_like(q)
    cu = torch.tensor([0, 1 << 20], dtype=torch.int32, device="cuda")
    prompt_attention(q, k, v, out, cu, 64, 0.1)
    assert torch.equal(out, want)
    out = torch.full_like(q, 2.0)
    prompt_attention(q, k, v, out, torch.tensor([-5, -3], dtype=torch.int32, device="cuda"), 64, 0.1)
    assert (out == 2.0).all()
    # Rows that several sequences share would be more work than the call has room for: dropped.
    cu = torch.tensor([0, 64, 0, 64, 0, 64], dtype=torch.int32, device="cuda")
    prompt_attention(q, k, v, torch.empty_like(q), cu, 64, 0.1)
    torch.cuda.synchronize()
    assert _lib.device_error() == _lib.DEVERR_NONE


def test_matches_the_paged_kernel():
    """The same batch through a cache: both are the same attention, within both roundings."""
    L = [96, 208]
    q, k, v = _inputs(L, L, 16, 2, 128, torch.bfloat16, 9)
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    prompt_attention(q.cuda(), k.cuda(), v.cuda(), out, _cu(L).cuda(), 208, 128 ** -0.5)
    kc, vc = k.view(-1, 16, 2, 128).cuda(), v.view(-1, 16, 2, 128).cuda()
    table = torch.tensor([list(range(6)) + [0] * 7, list(range(6, 19))], dtype=torch.int32, device="cuda")
    paged = torch.empty_like(out)
    paged_split_kv_attention(q.cuda(), kc, vc, paged, table, torch.tensor(L, dtype=torch.int32, device="cuda"),
                             _cu(L).cuda(), 208, 208, 128 ** -0.5, num_splits=1)
    assert (out.float() - paged.float()).abs().max().item() <= 2 * 2 ** -8 * out.float().abs().max().item()


def test_streams_graph_and_threads():
    ql = [150, 61]
    q, k, v = _inputs(ql, ql, 8, 2, 128, torch.bfloat16, 12)
    qg, kg, vg, cu = q.cuda(), k.cuda(), v.cuda(), _cu(ql).cuda()
    want = torch.empty_like(qg)
    prompt_attention(qg, kg, vg, want, cu, 150, 0.1)
    torch.cuda.synchronize()
    # Another stream than the tensors' own.
    side = torch.cuda.Stream()
    out = torch.empty_like(qg)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prompt_attention(qg, kg, vg, out, cu, 150, 0.1)
    side.synchronize()
    assert torch.equal(out, want)
    # Two captured calls, replayed at the same time on two streams with an eager call between.
    outs = [torch.zeros_like(qg) for _ in range(2)]
    graphs = []
    for o in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            prompt_attention(qg, kg, vg, o, cu, 150, 0.1)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        prompt_attention(qg, kg, vg, out, cu, 150, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all(torch.equal(o, want) for o in outs)
    # Threads that launch on one stream at once: no call reads another's work list.
    results = [torch.empty_like(qg) for _ in range(4)]

    def work(o):
        for _ in range(30):
            prompt_attention(qg, kg, vg, o, cu, 150, 0.1)

    threads = [threading.Thread(target=work, args=(o,)) for o in results]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in results)
    assert _lib.device_error() == _lib.DEVERR_NONE
