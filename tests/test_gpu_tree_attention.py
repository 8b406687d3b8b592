"""Draft-tree attention against its 64-bit definition (GPU): types, head shapes, page sizes,
trees of one node to more than a tile, masks that leave a row empty, bad page tails, tables
and lengths, streams, graphs, and the routes that reach it."""

from __future__ import annotations

import random

import pytest
import torch

from minicpm_b200 import _lib, iluvatar_attention, paged_split_kv_attention, paged_tree_attention
from oracle import attention_tolerance, tree_attention_reference

pytestmark = pytest.mark.gpu


def tree_masks(nodes, width, rng):
    """Random trees, parents first: row i sees its ancestors and itself."""
    mask = torch.zeros(sum(nodes), width, dtype=torch.bool)
    row = 0
    for n in nodes:
        for i in range(n):
            parent = rng.randint(-1, i - 1)
            if parent >= 0:
                mask[row + i] = mask[row + parent]
            mask[row + i, i] = True
        row += n
    return mask


class Batch:
    def __init__(self, ctx, nodes, hq=16, hkv=2, dim=128, page=16, dtype=torch.bfloat16, seed=0, extra_pages=3,
                 extra_cols=0, width=None):
        g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
        self.nodes, self.lens = nodes, [c + n for c, n in zip(ctx, nodes)]
        need = [-(-L // page) for L in self.lens]
        pool = sum(need) + extra_pages
        ids = list(range(pool))
        rng.shuffle(ids)
        cols = max(need) + extra_cols
        rows, at = [], 0
        for n in need:
            rows.append(ids[at:at + n] + [ids[-1]] * (cols - n))
            at += n
        self.table = torch.tensor(rows, dtype=torch.int32)
        self.free = ids[at:]
        self.q = torch.randn(sum(nodes), hq, dim, generator=g).to(dtype)
        self.cache = torch.randn(pool, 2, page, hkv, dim, generator=g).to(dtype)
        self.mask = tree_masks(nodes, width or max(nodes + [1]), rng)
        self.cu = torch.tensor([0, *torch.tensor(nodes).cumsum(0).tolist()], dtype=torch.int32)
        self.page, self.dim, self.scale = page, dim, dim ** -0.5

    def run(self, cache=None, out=None, mask=None, **over):
        cache = self.cache.cuda() if cache is None else cache
        out = torch.full(self.q.shape, float("nan"), dtype=self.q.dtype, device="cuda") if out is None else out
        args = dict(tree_mask=(self.mask if mask is None else mask).cuda(), block_table=self.table.cuda(),
                    seqused_k=torch.tensor(self.lens, dtype=torch.int32).cuda(), cu_seqlens_q=self.cu.cuda(),
                    max_seqlen_q=max(self.nodes), max_seqlen_k=max(self.lens), softmax_scale=self.scale)
        args.update(over)
        got = paged_tree_attention(self.q.cuda(), cache[:, 0], cache[:, 1], out, **args)
        assert got is out
        torch.cuda.synchronize()
        return out

    def check(self, out, mask=None, tag=""):
        o, a, s = tree_attention_reference(self.q, self.cache[:, 0], self.cache[:, 1], self.mask if mask is None else mask,
                                           self.table, self.lens, self.cu.tolist(), self.scale)
        tol = attention_tolerance(o, a, s, max(self.lens), self.dim, self.q.dtype, self.cache.double().abs().max().item())
        d = (out.cpu().double() - o).abs()
        assert torch.isfinite(d).all(), f"{tag}: non-finite output"
        worst = (d / tol).max().item()
        assert worst <= 1.0, f"{tag}: {worst:.2f} of the bound"
        assert _lib.device_error() == _lib.DEVERR_NONE


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_types_and_head_dims(dim, dtype):
    b = Batch([100, 0, 517, 30], [16, 5, 31, 1], hq=8, dim=dim, dtype=dtype, seed=dim)
    b.check(b.run())


@pytest.mark.parametrize("hq,hkv", [(16, 2), (4, 4), (9, 9), (16, 16), (6, 1), (24, 8), (128, 1), (40, 4)])
def test_head_groups(hq, hkv):
    b = Batch([90, 260], [13, 40], hq=hq, hkv=hkv, dim=64, seed=hq)
    b.check(b.run())


@pytest.mark.parametrize("page", [16, 32, 48, 128, 256])
def test_page_sizes(page):
    b = Batch([15, 300, 1], [17, 33, 2], page=page, seed=page)
    b.check(b.run())


@pytest.mark.parametrize("page", [32, 64, 128, 384])
@pytest.mark.parametrize("dim,hq,hkv", [(64, 9, 9), (128, 12, 12), (256, 10, 10), (64, 4, 2), (256, 4, 2)])
def test_larger_slices(page, dim, hq, hkv):
    """Pages of 32 keys and more come in larger boxes, through one map per head and through one for all."""
    b = Batch([129, 5, 600], [9, 21, 3], hq=hq, hkv=hkv, dim=dim, page=page, seed=page + dim)
    cache = b.cache.clone()
    for row, L in enumerate(b.lens):  # the rest of every last page may hold anything
        if L % page:
            cache[int(b.table[row, L // page]), :, L % page:] = float("nan")
    b.check(b.run(cache=cache.cuda()))


@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 17, 63, 64, 65, 128, 200])
@pytest.mark.parametrize("hq", [2, 16])
def test_trees_around_the_tiles(nodes, hq):
    # Contexts that put the first drafted key before, at and behind a tile's edge.
    b = Batch([128 - nodes % 128, 127, 128, 0, 129], [nodes] * 5, hq=hq, hkv=2, dim=64, seed=nodes)
    b.check(b.run(), tag=f"{nodes} {hq}")


def test_long_contexts_are_split_and_combined():
    for ctx, n, dim, dtype in (([9000], 16, 128, torch.bfloat16), ([20000, 5], 3, 64, torch.float16),
                               ([4090], 40, 256, torch.bfloat16)):
        b = Batch(ctx, [n] * len(ctx), hq=8, hkv=2, dim=dim, dtype=dtype, seed=n)
        b.check(b.run(), tag=f"{ctx} {n} {dim}")


@pytest.mark.parametrize("n", [64, 65, 400])
def test_many_sequences(n):
    r = random.Random(n)
    b = Batch([r.randrange(40) for _ in range(n)], [r.randrange(6) for _ in range(n)], hq=4, hkv=2, dim=64, seed=n)
    b.check(b.run())


@pytest.mark.parametrize("hint", [1, 600, 1 << 20])
def test_a_wrong_bound_of_the_longest_sequence_costs_time_only(hint):
    b = Batch([2100, 33], [9, 40], hq=8, hkv=1, seed=3)
    b.check(b.run(max_seqlen_k=hint))


def test_masks_that_leave_rows_empty_and_unseen_garbage():
    """A row that sees nothing is 0; K/V of tokens past the length may be NaN; so may tail pages."""
    b = Batch([0, 40, 0], [20, 9, 3], seed=3)
    mask = b.mask.clone()
    mask[4] = False
    mask[29:] = False
    mask[22] = False  # still sees the context
    cache = b.cache.clone()
    for row, L in enumerate(b.lens):
        if L % 16:
            cache[int(b.table[row, L // 16]), :, L % 16:] = float("nan")
    for p in b.free:
        cache[p] = float("nan")
    out = b.run(cache=cache.cuda(), mask=mask)
    b.check(out, mask=mask)
    assert out[4].abs().max().item() == 0.0 and out[29:].abs().max().item() == 0.0


@pytest.mark.parametrize("hq,hkv,dim", [(16, 2, 128), (16, 2, 64), (2, 2, 128), (16, 2, 256), (12, 12, 64)])
@pytest.mark.parametrize("nodes", [5, 20, 100, 150])
def test_drafted_tokens_that_nobody_sees_may_hold_anything(hq, hkv, dim, nodes):
    """A padded draft: slots whose K/V rows were never written (NaN) are hidden from every row."""
    b = Batch([0, 119, 128, 1000], [nodes] * 4, hq=hq, hkv=hkv, dim=dim, seed=nodes)
    r, mask, cache = random.Random(nodes), b.mask.clone(), b.cache.clone()
    for row, L in enumerate(b.lens):
        for j in r.sample(range(nodes), nodes // 3) + [nodes - 1]:
            mask[row * nodes:(row + 1) * nodes, j] = False
            pos = L - nodes + j
            cache[int(b.table[row, pos // b.page]), :, pos % b.page] = float("nan")
    out = b.run(cache=cache.cuda(), mask=mask)
    b.check(out, mask=mask)


def test_any_mask_goes():
    b = Batch([37, 200], [30, 61], seed=11, width=70)
    mask = torch.rand(b.mask.shape, generator=torch.Generator().manual_seed(1)) < 0.4
    b.check(b.run(mask=mask), mask=mask)
    b.check(b.run(mask=mask.to(torch.uint8) * 255), mask=mask)
    wide = torch.zeros(mask.shape[1], mask.shape[0], dtype=torch.bool)
    wide.copy_(mask.t())
    b.check(b.run(mask=wide.t()), mask=mask)  # columns not contiguous


def test_more_drafted_tokens_than_keys():
    b = Batch([0, 0], [12, 7], seed=2)
    b.lens = [5, 7]
    b.check(b.run())


def test_lower_triangular_mask_is_causal_attention_and_one_token_is_decode():
    b = Batch([300, 64, 1000], [24, 24, 24], seed=21)
    mask = torch.tril(torch.ones(24, 24, dtype=torch.bool)).repeat(3, 1)
    out = b.run(mask=mask)
    b.check(out, mask=mask)
    c = b.cache.cuda()
    paged = torch.empty_like(out)
    lens = torch.tensor(b.lens, dtype=torch.int32).cuda()
    paged_split_kv_attention(b.q.cuda(), c[:, 0], c[:, 1], paged, b.table.cuda(), lens, b.cu.cuda(), 24, max(b.lens),
                             b.scale, num_splits=1)
    assert (out.float() - paged.float()).abs().max().item() <= 2 * 2 ** -8 * out.float().abs().max().item()
    one = Batch([511, 16, 0], [1, 1, 1], seed=22)
    one.check(one.run())


def test_empty_requests_int64_and_rows_behind():
    b = Batch([40, 7, 90], [6, 0, 11], seed=5, extra_cols=4)
    q = torch.randn(20, 16, 128).to(torch.bfloat16)
    q[:17] = b.q
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device="cuda")
    c, mask = b.cache.cuda(), torch.zeros(20, 11, dtype=torch.bool)
    mask[:17] = b.mask
    paged_tree_attention(q.cuda(), c[:, 0], c[:, 1], out, mask.cuda(), b.table.long().cuda(),
                         torch.tensor(b.lens).cuda(), b.cu.long().cuda(), 11, max(b.lens), b.scale)
    b.check(out[:17])
    assert (out[17:] == 5.0).all()


def test_bad_pages_and_lengths_stay_in_bounds():
    b = Batch([100], [8], seed=6)
    table = b.table.clone()
    table[0, 1], table[0, 2] = 1 << 30, -7
    out = b.run(block_table=table.cuda())
    assert torch.isfinite(out.float()).all()  # such a page reads as zeros
    far = table.long()
    far[0, 1], far[0, 2] = (1 << 32) + 1, -(1 << 32)
    assert torch.equal(b.run(block_table=far.cuda()), out)
    want = b.run()
    out = b.run(seqused_k=torch.tensor([1 << 30], dtype=torch.int32).cuda())  # clipped to the table's pages
    assert torch.isfinite(out.float()).all() and out.shape == want.shape
    wide = dict(cu_seqlens_q=b.cu.long().cuda())
    far = b.run(seqused_k=torch.tensor([(1 << 32) + 108]).cuda(), **wide)  # not 108
    assert torch.equal(far, out)
    out = b.run(seqused_k=torch.tensor([-4], dtype=torch.int32).cuda())
    assert out.abs().max().item() == 0.0
    out = b.run(cu_seqlens_q=torch.tensor([0, 1 << 29], dtype=torch.int32).cuda())
    assert torch.isfinite(out.float()).all()
    assert _lib.device_error() == _lib.DEVERR_NONE


def test_split_views_of_another_layout():
    b = Batch([77, 5], [9, 14], hq=8, hkv=2, seed=8)
    hnd = b.cache.permute(0, 1, 3, 2, 4).contiguous().cuda().permute(0, 1, 3, 2, 4)  # heads outermost in memory
    b.check(b.run(cache=hnd))


def test_graph_and_streams():
    b = Batch([500, 33], [12, 12], seed=13)
    want = b.run()
    c = b.cache.cuda()
    args = (b.mask.cuda(), b.table.cuda(), torch.tensor(b.lens, dtype=torch.int32).cuda(), b.cu.cuda(), 12, max(b.lens),
            b.scale)
    q = b.q.cuda()
    outs, graphs = [torch.zeros_like(want) for _ in range(2)], []
    for o in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_tree_attention(q, c[:, 0], c[:, 1], o, *args)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    eager = torch.empty_like(want)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        paged_tree_attention(q, c[:, 0], c[:, 1], eager, *args)
    torch.cuda.synchronize()
    assert torch.equal(eager, want) and all(torch.equal(o, want) for o in outs)


def test_same_call_gives_the_same_bits():
    b = Batch([7000, 300, 20], [16, 7, 33], seed=17)
    first = b.run()
    assert all(torch.equal(first, b.run()) for _ in range(5))
