"""Page operators of the cache against a plain restatement (GPU): element types, layouts,
page sizes, one to many sequences, indices named twice, what cannot be served, graphs."""

from __future__ import annotations

import random

import pytest
import torch

from minicpm_b200 import _lib, kv_pages

pytestmark = pytest.mark.gpu


def _caches(layers, pool, page, heads, dim, dtype, seed=0, hnd=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(layers):
        shape = (pool, 2, heads, page, dim) if hnd else (pool, 2, page, heads, dim)
        t = torch.randint(0, 256, (*shape, torch.empty(0, dtype=dtype).element_size()), generator=g, dtype=torch.uint8)
        t = t.view(dtype).view(shape)
        out.append(t.permute(0, 1, 3, 2, 4) if hnd else t)
    return out


def _views(cache):
    return [cache[:, 0], cache[:, 1]]


def _layers(caches, split=False):
    gpu = []
    for c in caches:
        if c.is_contiguous():
            gpu.append(c.cuda())
        else:
            gpu.append(c.permute(0, 1, 3, 2, 4).contiguous().cuda().permute(0, 1, 3, 2, 4))
    flat = [v for c in gpu for v in _views(c)] if split else gpu
    return gpu, kv_pages.cache_layers(flat)


def _bits(t):
    return t.contiguous().view(torch.uint8)


def _same(gpu, cpu):
    assert all(torch.equal(_bits(g.cpu()), _bits(c)) for g, c in zip(gpu, cpu))


KINDS = [(torch.bfloat16, 128, False), (torch.float16, 64, True), (torch.float8_e4m3fn, 132, False),
         (torch.int8, 68, True), (torch.float32, 64, False)]


@pytest.mark.parametrize("dtype,dim,hnd", KINDS)
@pytest.mark.parametrize("page", [16, 48])
def test_copy_pages(dtype, dim, hnd, page):
    caches = _caches(3, 37, page, 2, dim, dtype, hnd=hnd)
    gpu, layers = _layers(caches, split=hnd)
    src, dst = [3, 0, 3, -1, 9, 11], [20, 36, 21, 5, -2, 11]
    kv_pages.copy_pages(layers, torch.tensor(src).cuda(), torch.tensor(dst).cuda())
    for c in caches:
        c[[20, 36, 21]] = c[[3, 0, 3]]
    _same(gpu, caches)
    assert _lib.device_error() == _lib.DEVERR_NONE
    kv_pages.copy_pages(gpu, torch.tensor([37, 1], dtype=torch.int32).cuda(), torch.tensor([2, 1 << 20], dtype=torch.int32).cuda())
    _same(gpu, caches)
    assert _lib.device_error() == _lib.DEVERR_PAGE_RANGE


def test_copy_many_pages_and_layers():
    caches = _caches(128, 64, 16, 1, 64, torch.bfloat16, seed=4)
    gpu, layers = _layers(caches)
    perm = torch.randperm(64, generator=torch.Generator().manual_seed(2))
    kv_pages.copy_pages(layers, perm[:31].cuda(), perm[32:63].cuda())
    for c in caches:
        c[perm[32:63]] = c[perm[:31]]
    _same(gpu, caches)


class Pool:
    """The plain restatement of the pool, on the CPU."""

    def __init__(self, lens, spare, page, pool, cols, caches, dtype=torch.int32, seed=0):
        rng = random.Random(seed)
        ids = list(range(pool))
        rng.shuffle(ids)
        self.page, self.pool = page, pool
        self.table, self.lens, self.refs = [], list(lens) + [0] * spare, [0] * pool
        at = 0
        for n in self.lens:
            need = -(-n // page)
            self.table.append(ids[at:at + need] + [-1] * (cols - need))
            at += need
        for row in self.table:
            for p in row:
                if p >= 0:
                    self.refs[p] += 1
        self.caches = caches
        self.dtype = dtype

    def gpu(self):
        return (torch.tensor(self.table, dtype=self.dtype).cuda(), torch.tensor(self.lens, dtype=self.dtype).cuda(),
                torch.tensor(self.refs, dtype=torch.int32).cuda())

    def fork(self, parents, children):
        before, lens = [r[:] for r in self.table], self.lens[:]
        plan = []
        claimed = set()
        for p, c in zip(parents, children):
            if p < 0 or c < 0 or p >= len(lens) or c >= len(lens):
                continue
            first = c not in claimed
            claimed.add(c)
            if first and lens[c] == 0:
                plan.append((p, c))
        free = [i for i in range(self.pool) if self.refs[i] == 0]
        for p, c in plan:
            full, tail = divmod(lens[p], self.page)
            fresh = None
            if tail:
                if not free:
                    continue
                fresh = free.pop(0)
                self.refs[fresh] = 1
                for t in self.caches:
                    t[fresh, :, :tail] = t[before[p][full], :, :tail]
            row = before[p][:full] + ([fresh] if tail else [])
            for q in row[:full]:
                self.refs[q] += 1
            self.table[c] = row + [-1] * (len(before[p]) - len(row))
            self.lens[c] = lens[p]

    def free(self, rows):
        for r in rows:
            if 0 <= r < len(self.table):
                for p in self.table[r]:
                    if p >= 0:
                        self.refs[p] -= 1
                self.table[r] = [-1] * len(self.table[r])
                self.lens[r] = 0

    def check(self, table, lens, refs, gpu):
        torch.cuda.synchronize()
        assert lens.tolist() == self.lens
        assert table.tolist() == self.table
        assert refs.tolist() == self.refs
        _same(gpu, self.caches)


@pytest.mark.parametrize("dtype,dim,hnd", KINDS)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_fork_and_free(dtype, dim, hnd, index):
    caches = _caches(2, 60, 16, 2, dim, dtype, seed=1, hnd=hnd)
    pool = Pool([100, 1, 32, 0, 47], 6, 16, 60, 9, caches, index, seed=3)
    gpu, layers = _layers(caches, split=hnd)
    table, lens, refs = pool.gpu()
    steps = [([0, 0, 4, 2, 1, 3], [5, 6, 7, 8, 9, 10]), ([5, 7, 0], [10, 3, -1])]
    for parents, children in steps:
        kv_pages.fork_sequences(layers, table, lens, refs, torch.tensor(parents, dtype=index).cuda(),
                                torch.tensor(children, dtype=index).cuda())
        pool.fork(parents, children)
        pool.check(table, lens, refs, gpu)
    rows = [0, 6, 6, 3, -1, 2]
    kv_pages.free_sequences(table, lens, refs, torch.tensor(rows, dtype=index).cuda())
    pool.free(rows)
    pool.check(table, lens, refs, gpu)
    kv_pages.fork_sequences(layers, table, lens, refs, torch.tensor([7, 5], dtype=index).cuda(),
                            torch.tensor([0, 2], dtype=index).cuda())
    pool.fork([7, 5], [0, 2])
    pool.check(table, lens, refs, gpu)
    assert _lib.device_error() == _lib.DEVERR_NONE


def test_fork_errors_leave_the_rest_served():
    caches = _caches(1, 8, 16, 1, 64, torch.bfloat16)
    pool = Pool([20, 33], 5, 16, 8, 4, caches)  # 5 pages used, 3 free
    gpu, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    parents, children = [0, 0, 99, 0, 1, 1, 1], [2, 2, 3, 1, 3, 4, 5]
    kv_pages.fork_sequences(layers, table, lens, refs, torch.tensor(parents).cuda(), torch.tensor(children).cuda())
    pool.fork(parents, children)  # row 2 once, a row past the table, a row in use, then one page too few
    pool.check(table, lens, refs, gpu)
    assert pool.lens[5] == 0 and pool.lens[4] == 33
    assert _lib.device_error() in (_lib.DEVERR_SEQ_ROW, _lib.DEVERR_NO_PAGE)
    kv_pages.free_sequences(table, lens, refs, torch.tensor([70, 4]).cuda())
    pool.free([4])
    pool.check(table, lens, refs, gpu)
    assert _lib.device_error() == _lib.DEVERR_SEQ_ROW
    refs[int(table[0, 0])] = 0  # a count that is wrong does not go below zero
    kv_pages.free_sequences(table, lens, refs, torch.tensor([0]).cuda())
    assert refs.min().item() == 0
    assert _lib.device_error() == _lib.DEVERR_PAGE_RANGE


def test_fork_of_a_bad_table_is_refused():
    caches = _caches(1, 8, 16, 1, 64, torch.bfloat16)
    pool = Pool([20], 2, 16, 8, 4, caches)
    _, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    table[0, 1] = 1 << 20
    kv_pages.fork_sequences(layers, table, lens, refs, torch.tensor([0]).cuda(), torch.tensor([1]).cuda())
    assert lens.tolist() == [20, 0, 0] and _lib.device_error() == _lib.DEVERR_PAGE_RANGE
    lens[0] = 1000  # more than the row's columns hold
    kv_pages.fork_sequences(layers, table, lens, refs, torch.tensor([0]).cuda(), torch.tensor([1]).cuda())
    assert lens.tolist() == [1000, 0, 0] and _lib.device_error() == _lib.DEVERR_SEQ_ROW


def test_a_large_fork():
    """More entries than the planning block has threads, a pool past one of its passes."""
    n = 1300
    caches = _caches(1, 9000, 16, 1, 64, torch.bfloat16, seed=6)
    pool = Pool([77, 160, 31], n, 16, 9000, 11, caches, seed=8)
    gpu, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    r = random.Random(1)
    parents, children = [r.randrange(3) for _ in range(n)], list(range(3, n + 3))
    r.shuffle(children)
    kv_pages.fork_sequences(layers, table, lens, refs, torch.tensor(parents).cuda(), torch.tensor(children).cuda())
    pool.fork(parents, children)
    pool.check(table, lens, refs, gpu)
    kv_pages.free_sequences(table, lens, refs, torch.tensor(children).cuda())
    pool.free(children)
    pool.check(table, lens, refs, gpu)
    assert _lib.device_error() == _lib.DEVERR_NONE


def _keep_plain(caches, table, context, accepted, counts, page):
    for b, c in enumerate(context):
        for i in range(counts[b]):
            a = c + accepted[b][i]
            for t in caches:
                t[table[b][(c + i) // page], :, (c + i) % page] = t[table[b][a // page], :, a % page].clone()


@pytest.mark.parametrize("dtype,dim,hnd", KINDS)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_keep_accepted_tokens(dtype, dim, hnd, index):
    page, draft = 16, 40
    context, counts = [0, 15, 16, 100, 37], [0, 1, 12, 40, 17]
    r = random.Random(5)
    accepted = [sorted(r.sample(range(draft), n)) + [-9] * (40 - n) for n in counts]
    caches = _caches(3, 64, page, 2, dim, dtype, seed=9, hnd=hnd)
    pool = Pool([c + draft for c in context], 0, page, 64, 10, caches, index, seed=2)
    gpu, layers = _layers(caches, split=hnd)
    table, lens, refs = pool.gpu()
    ctx = torch.tensor(context, dtype=index).cuda()
    acc, num = torch.tensor(accepted, dtype=index).cuda(), torch.tensor(counts, dtype=index).cuda()
    kv_pages.keep_accepted_tokens(layers, table, ctx, acc, num, lens)
    _keep_plain(caches, pool.table, context, accepted, counts, page)
    pool.lens = [c + n for c, n in zip(context, counts)]
    pool.check(table, lens, refs, gpu)
    kv_pages.keep_accepted_tokens(layers, table, ctx, torch.arange(40, device="cuda", dtype=index).repeat(5, 1), num, lens, refs)
    for b, n in enumerate(pool.lens):  # nothing moves, the pages behind are released
        for col in range(-(-n // page), 10):
            if pool.table[b][col] >= 0:
                pool.refs[pool.table[b][col]] -= 1
                pool.table[b][col] = -1
    pool.check(table, lens, refs, gpu)
    assert _lib.device_error() == _lib.DEVERR_NONE


def test_keep_refuses_bad_paths():
    page = 16
    caches = _caches(2, 40, page, 1, 64, torch.bfloat16, seed=3)
    pool = Pool([30] * 6, 0, page, 40, 3, caches)
    gpu, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    ctx = torch.tensor([10, 10, 10, 10, -1, 10], dtype=torch.int32).cuda()
    acc = torch.tensor([[1, 3, 2, 9], [1, 50, 51, 52], [2, 5, 6, 7], [-1, 2, 3, 4], [0, 1, 2, 3], [3, 4, 5, 6]], dtype=torch.int32)
    num = torch.tensor([4, 4, 9, 2, 2, -3], dtype=torch.int32)
    want = [2, 1, 4, 0, 0, 0]
    kv_pages.keep_accepted_tokens(layers, table, ctx, acc.cuda(), num.cuda(), lens)
    _keep_plain(caches, pool.table, [10, 10, 10, 10, 0, 10], acc.tolist(), want, page)
    pool.lens = [12, 11, 14, 10, 0, 10]
    pool.check(table, lens, refs, gpu)
    assert _lib.device_error() in (_lib.DEVERR_ACCEPT, _lib.DEVERR_PAGE_RANGE)


@pytest.mark.parametrize("index,bad", [(torch.int32, -1), (torch.int64, -(1 << 40)), (torch.int64, 1 << 40)])
def test_keep_leaves_the_pages_of_a_bad_context(index, bad):
    page = 16
    caches = _caches(1, 12, page, 1, 64, torch.bfloat16, seed=3)
    pool = Pool([40, 50], 0, page, 12, 4, caches, index)
    gpu, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    ctx = torch.tensor([bad, 30], dtype=index).cuda()
    acc, num = torch.tensor([[0, 1], [0, 1]], dtype=index).cuda(), torch.tensor([2, 2], dtype=index).cuda()
    kv_pages.keep_accepted_tokens(layers, table, ctx, acc, num, lens, refs)
    pool.lens = [0, 32]  # row 0 still names its pages; row 1 gives back the two behind 32 tokens
    for col in (2, 3):
        pool.refs[pool.table[1][col]] -= 1
        pool.table[1][col] = -1
    pool.check(table, lens, refs, gpu)
    assert _lib.device_error() == _lib.DEVERR_ACCEPT
    kv_pages.free_sequences(table, lens, refs, torch.tensor([0]).cuda())
    assert (table[0] == -1).all() and refs.sum().item() == 2


def test_fork_of_a_parent_that_lacks_a_full_page():
    caches = _caches(1, 8, 16, 1, 64, torch.bfloat16)
    pool = Pool([40], 2, 16, 8, 4, caches)
    _, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    table[0, 0] = -1
    kv_pages.fork_sequences(layers, table, lens, refs, torch.tensor([0]).cuda(), torch.tensor([1]).cuda())
    row = table[1].tolist()
    assert row[0] == -1 and row[1] == int(table[0, 1]) and row[2] >= 0 and row[3] == -1
    assert refs[row[1]].item() == 2 and refs[row[2]].item() == 1 and _lib.device_error() == _lib.DEVERR_PAGE_RANGE


def test_keep_does_not_write_shared_pages():
    page = 16
    caches = _caches(1, 12, page, 1, 64, torch.bfloat16, seed=3)
    pool = Pool([40, 0], 0, page, 12, 4, caches)
    gpu, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    kv_pages.fork_sequences(layers, table, lens, refs, torch.tensor([0]).cuda(), torch.tensor([1]).cuda())
    pool.fork([0], [1])
    ctx = torch.tensor([20, 34], dtype=torch.int32).cuda()  # row 0 would write the page that row 1 shares
    acc = torch.tensor([[0, 1, 5], [1, 2, 4]], dtype=torch.int32).cuda()
    num = torch.tensor([3, 3], dtype=torch.int32).cuda()
    kv_pages.keep_accepted_tokens(layers, table, ctx, acc, num, lens, refs)
    _keep_plain(caches, pool.table, [20, 34], acc.tolist(), [2, 3], page)
    pool.lens = [22, 37]
    pool.refs[pool.table[0][2]] -= 1
    pool.table[0][2] = -1
    pool.check(table, lens, refs, gpu)
    assert _lib.device_error() == _lib.DEVERR_PAGE_SHARED


def test_graph_replays_a_step_of_a_search():
    """free + fork captured once and replayed: the indices are read at every replay."""
    caches = _caches(2, 64, 16, 2, 64, torch.bfloat16, seed=7)
    pool = Pool([90, 41], 4, 16, 64, 8, caches, seed=1)
    gpu, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    parents = torch.tensor([0, 1, 0, 1], dtype=torch.int32).cuda()
    children = torch.tensor([2, 3, 4, 5], dtype=torch.int32).cuda()

    def step():
        kv_pages.free_sequences(table, lens, refs, children)
        kv_pages.fork_sequences(layers, table, lens, refs, parents, children)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for order in ([0, 1, 0, 1], [1, 1, 1, 0], [-1, 0, 0, 1]):
        parents.copy_(torch.tensor(order, dtype=torch.int32))
        graph.replay()
        pool.free([2, 3, 4, 5])
        pool.fork(order, [2, 3, 4, 5])
        pool.check(table, lens, refs, gpu)
    assert _lib.device_error() == _lib.DEVERR_NONE
