"""The serving operators together, as a speculative decoder with branches uses them (GPU).

A batch of prompts goes through ``prompt_attention`` and into the paged cache; then, step after
step, drafted trees are written behind the contexts, attended (service, dispatcher and operator
alike), the accepted paths are kept, and sequences are forked and freed.  Beside it runs a plain
model of every sequence: the list of its K/V rows.  Attention is held to 64 bits on those lists,
the cache to their bits.
"""

from __future__ import annotations

import random
from types import SimpleNamespace

import pytest
import torch

from minicpm_b200 import _lib, iluvatar_attention, kv_pages, paged_tree_attention, prompt_attention, service
from minicpm_b200.kv_cache import reshape_and_cache_flash
from oracle import attention_tolerance
from oracle.varlen_attention import attend
from test_gpu_tree_attention import tree_masks

pytestmark = pytest.mark.gpu

HQ, HKV, DIM, PAGE, LAYERS, POOL, COLS, ROWS = 8, 2, 128, 16, 3, 160, 14, 8


def _check(got, want, keys, dtype, v_max):
    o, a, s = want
    d = (got.cpu().double() - o).abs()
    assert (d / attention_tolerance(o, a, s, keys, DIM, dtype, v_max)).max().item() <= 1.0


class Decoder:
    def __init__(self, dtype):
        self.dtype, self.g, self.rng = dtype, torch.Generator().manual_seed(4), random.Random(4)
        self.caches = [torch.zeros(POOL, 2, PAGE, HKV, DIM, dtype=dtype, device="cuda") for _ in range(LAYERS)]
        self.layers = kv_pages.cache_layers(self.caches)
        self.table = torch.full((ROWS, COLS), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(ROWS, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(POOL, dtype=torch.int32, device="cuda")
        self.model = {}  # row -> [layers, 2, length, HKV, DIM]

    def rows(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype)

    def grow(self, row, new):
        """The scheduler's part: pages for `new` more tokens, and their slots."""
        table, refs, length = self.table.cpu(), self.refs.cpu(), int(self.lens[row])
        slots = []
        for pos in range(length, length + new):
            if table[row, pos // PAGE] < 0:
                page = int((refs == 0).nonzero()[0])
                refs[page], table[row, pos // PAGE] = 1, page
            slots.append(int(table[row, pos // PAGE]) * PAGE + pos % PAGE)
        self.table.copy_(table)
        self.refs.copy_(refs)
        return slots

    def write(self, slots, kv):
        """K/V rows [layers, 2, tokens, HKV, DIM] at their slots."""
        one = torch.ones(1, device="cuda")
        for c, (k, v) in zip(self.caches, kv.cuda()):
            reshape_and_cache_flash(k, v, c[:, 0], c[:, 1], torch.tensor(slots).cuda(), "auto", one, one)

    def cached(self, row):
        L = int(self.lens[row])
        pages = self.table[row, :-(-L // PAGE)].long()
        return torch.stack([c[pages].transpose(0, 1).reshape(2, -1, HKV, DIM)[:, :L].cpu() for c in self.caches])

    def check(self):
        torch.cuda.synchronize()
        refs = torch.zeros(POOL, dtype=torch.int32)
        for row in range(ROWS):
            want = self.model.get(row)
            assert int(self.lens[row]) == (0 if want is None else want.shape[2])
            if want is not None:
                assert torch.equal(self.cached(row), want)
            for p in self.table[row].tolist():
                if p >= 0:
                    refs[p] += 1
        assert torch.equal(refs, self.refs.cpu())
        assert _lib.device_error() == _lib.DEVERR_NONE


def _tree_step(d, live, monkeypatch):
    nodes = [d.rng.randint(1, 20) for _ in live]
    mask = tree_masks(nodes, max(nodes), d.rng)
    drafts = [d.rows(LAYERS, 2, n, HKV, DIM) for n in nodes]
    slots = [s for row, n in zip(live, nodes) for s in d.grow(row, n)]
    d.write(slots, torch.cat(drafts, dim=2))
    context = d.lens[live].clone()
    total = context + torch.tensor(nodes, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, *torch.tensor(nodes).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    q, longest = d.rows(sum(nodes), HQ, DIM), int(total.max())
    table, scale, layer = d.table[live].clamp_min(0), DIM ** -0.5, LAYERS - 1
    cache = d.caches[layer]
    out = torch.empty(q.shape, dtype=d.dtype, device="cuda")
    paged_tree_attention(q.cuda(), cache[:, 0], cache[:, 1], out, mask.cuda(), table, total, cu, max(nodes), longest, scale)
    at = 0
    for row, n, draft in zip(live, nodes, drafts):
        kv = torch.cat([d.model[row], draft], dim=2)[layer]
        seen = torch.cat([torch.ones(n, kv.shape[1] - n, dtype=torch.bool), mask[at:at + n, :n]], dim=1)
        _check(out[at:at + n], attend(q[at:at + n], kv[0], kv[1], seen, scale), kv.shape[1], d.dtype, kv.double().abs().max().item())
        at += n
    # The same call through the dispatcher and through the service's layer: the same bits.
    monkeypatch.setenv("ILUVATAR_USE_OPTIMIZED", "1")
    monkeypatch.setenv("ILUVATAR_SPLIT_KV", "1")
    again = torch.empty_like(out)
    iluvatar_attention(q.cuda(), cache, cache, again, cu, max(nodes), total, longest, scale, block_table=table,
                       tree_mask=mask.cuda())
    assert torch.equal(again, out)
    impl = service.IluvatarAttentionImpl(HQ, DIM, scale, HKV, None, None, "auto")
    builder = service.IluvatarAttentionMetadataBuilder(HQ, HKV, DIM, torch.device("cuda"))
    meta = builder.build(0, SimpleNamespace(
        num_reqs=len(live), num_actual_tokens=sum(nodes), max_query_len=max(nodes), max_seq_len=longest, query_start_loc=cu,
        seq_lens=total, block_table_tensor=table, slot_mapping=None, causal=True, tree_mask=mask.cuda()))
    impl.forward(SimpleNamespace(), q.cuda(), q.cuda(), q.cuda(), cache, meta, again.zero_())
    assert torch.equal(again, out)
    # A path from the root in every tree is accepted.
    paths, at = [], 0
    for row, n, draft in zip(live, nodes, drafts):
        leaf = d.rng.randrange(n)
        path = mask[at + leaf, :n].nonzero().flatten().tolist()[:d.rng.randint(0, n)]
        paths.append(path)
        d.model[row] = torch.cat([d.model[row], draft[:, :, path]], dim=2)
        at += n
    most = max(1, *(len(p) for p in paths))
    table, lens = d.table[live], torch.zeros(len(live), dtype=torch.int32, device="cuda")
    kv_pages.keep_accepted_tokens(
        d.layers, table, context, torch.tensor([p + [-1] * (most - len(p)) for p in paths], dtype=torch.int32).cuda(),
        torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda(), lens, d.refs)
    d.table[live], d.lens[live] = table, lens
    d.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_drafts_and_branches(dtype, monkeypatch):
    d = Decoder(dtype)
    lens = [37, 16, 90]
    kv = [d.rows(LAYERS, 2, n, HKV, DIM) for n in lens]
    q = d.rows(sum(lens), HQ, DIM)
    packed = torch.cat(kv, dim=2).cuda()
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    out = torch.empty(q.shape, dtype=dtype, device="cuda")
    prompt_attention(q.cuda(), packed[0, 0], packed[0, 1], out, cu, max(lens), DIM ** -0.5)
    at = 0
    for row, (n, rows) in enumerate(zip(lens, kv)):
        seen = torch.tril(torch.ones(n, n, dtype=torch.bool))
        _check(out[at:at + n], attend(q[at:at + n], rows[0, 0], rows[0, 1], seen, DIM ** -0.5), n, dtype,
               rows.double().abs().max().item())
        at += n
        slots = d.grow(row, n)
        d.write(slots, rows)
        d.lens[row] = n
        d.model[row] = rows
    d.check()

    def fork(parents, children):
        kv_pages.fork_sequences(d.layers, d.table, d.lens, d.refs, torch.tensor(parents).cuda(), torch.tensor(children).cuda())
        for p, c in zip(parents, children):
            d.model[c] = d.model[p]
        d.check()

    def free(rows):
        kv_pages.free_sequences(d.table, d.lens, d.refs, torch.tensor(rows).cuda())
        for r in rows:
            d.model.pop(r, None)
        d.check()

    _tree_step(d, [0, 1, 2], monkeypatch)
    fork([0, 0, 2], [3, 4, 5])
    _tree_step(d, [0, 1, 2, 3, 4, 5], monkeypatch)
    free([1, 0, 2])
    fork([5, 3], [0, 1])
    for _ in range(3):
        _tree_step(d, sorted(d.model), monkeypatch)
    free(sorted(d.model))
    assert d.refs.abs().max().item() == 0 and (d.table == -1).all()


@pytest.mark.parametrize("kind", ["fp8", "int8_per_token_head"])
def test_trees_over_quantised_caches(kind, monkeypatch):
    """The service's quantised caches: pages dequantised, then the tree kernel; the oracle reads the dequantised rows."""
    from minicpm_b200.kv_cache import dequantize_kv_pages

    monkeypatch.setenv("ILUVATAR_USE_OPTIMIZED", "1")
    monkeypatch.setenv("ILUVATAR_SPLIT_KV", "1")
    rng, g = random.Random(2), torch.Generator().manual_seed(2)
    lens, nodes = [70, 33], [9, 14]
    impl = service.IluvatarAttentionImpl(HQ, DIM, DIM ** -0.5, HKV, None, None, kind)
    shape = service.IluvatarAttentionBackend.get_kv_cache_shape(12, PAGE, HKV, DIM, kind)
    cache = torch.zeros(shape, dtype=torch.int8 if kind.startswith("int8") else torch.uint8, device="cuda")
    scale = torch.full((1,), 0.05, device="cuda")
    layer = SimpleNamespace(_k_scale=scale, _v_scale=scale, _q_scale=scale)
    table = torch.tensor([[3, 0, 7, 5, 9], [1, 11, 4, 0, 0]], dtype=torch.int32)
    slots = [int(table[b, p // PAGE]) * PAGE + p % PAGE for b, L in enumerate(lens) for p in range(L)]
    k, v = (torch.randn(sum(lens), HKV, DIM, generator=g).to(torch.bfloat16) for _ in range(2))
    impl.do_kv_cache_update(layer, k.cuda(), v.cuda(), cache, torch.tensor(slots).cuda())
    mask = tree_masks(nodes, max(nodes), rng)
    q = torch.randn(sum(nodes), HQ, DIM, generator=g).to(torch.bfloat16)
    cu, total = torch.tensor([0, 9, 23], dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    builder = service.IluvatarAttentionMetadataBuilder(HQ, HKV, DIM, torch.device("cuda"))
    meta = builder.build(0, SimpleNamespace(
        num_reqs=2, num_actual_tokens=sum(nodes), max_query_len=max(nodes), max_seq_len=max(lens), query_start_loc=cu,
        seq_lens=total, block_table_tensor=table.cuda(), slot_mapping=None, causal=True, tree_mask=mask.cuda()))
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    impl.forward(layer, q.cuda(), q.cuda(), q.cuda(), cache, meta, out)
    kc, vc = impl._split_cache(cache)
    extra = dict(k_descale=scale, v_descale=scale) if kind == "fp8" else dict(k_scale_cache=impl._k_scale_cache,
                                                                             v_scale_cache=impl._v_scale_cache)
    dense, pages = dequantize_kv_pages(kc, vc, table.cuda(), total, max(lens), int(impl._kv_quant_mode), q.dtype, DIM, **extra)
    dense, pages, at = dense.cpu(), pages.cpu(), 0
    for b, (L, n) in enumerate(zip(lens, nodes)):
        rows = dense[pages[b, :-(-L // PAGE)].long()].transpose(0, 1).reshape(2, -1, HKV, DIM)[:, :L]
        seen = torch.cat([torch.ones(n, L - n, dtype=torch.bool), mask[at:at + n, :n]], dim=1)
        _check(out[at:at + n], attend(q[at:at + n], rows[0], rows[1], seen, DIM ** -0.5), L, q.dtype, rows.double().abs().max().item())
        at += n
    assert _lib.device_error() == _lib.DEVERR_NONE


@pytest.mark.parametrize("hq,hkv,dim", [(12, 12, 64), (16, 2, 128)])
def test_the_service_runs_encoder_batches(hq, hkv, dim, monkeypatch):
    monkeypatch.setenv("ILUVATAR_USE_OPTIMIZED", "1")
    monkeypatch.setenv("ILUVATAR_SPLIT_KV", "1")
    g, lens = torch.Generator().manual_seed(1), [50, 129, 3]
    q, k, v = (torch.randn(sum(lens) + 10, h, dim, generator=g).half() for h in (hq, hkv, hkv))
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    builder = service.IluvatarAttentionMetadataBuilder(hq, hkv, dim, torch.device("cuda"))
    meta = builder.build(0, SimpleNamespace(
        num_reqs=3, num_actual_tokens=sum(lens), max_query_len=129, max_seq_len=129, query_start_loc=cu.cuda(),
        seq_lens=torch.tensor(lens).cuda(), block_table_tensor=None, slot_mapping=None, causal=False))
    impl = service.IluvatarAttentionImpl(hq, dim, 0.11, hkv, None, None, "auto", attn_type=service.AttentionType.ENCODER)
    out = torch.full((sum(lens) + 10, hq, dim), 9.0, dtype=q.dtype, device="cuda")
    impl.forward(SimpleNamespace(), q.cuda(), k.cuda(), v.cuda(), torch.zeros(0), meta, out)
    at = 0
    for n in lens:
        rows = slice(at, at + n)
        want = attend(q[rows], k[rows], v[rows], torch.ones(n, n, dtype=torch.bool), 0.11)
        o, a, s = want
        d = (out[rows].cpu().double() - o).abs()
        assert (d / attention_tolerance(o, a, s, n, dim, q.dtype, v.double().abs().max().item())).max().item() <= 1.0
        at += n
    assert (out[sum(lens):] == 9.0).all()
