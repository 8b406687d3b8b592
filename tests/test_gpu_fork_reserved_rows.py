"""Forks into rows of length 0 that still name pages (GPU): the counts stay those of the table."""

from __future__ import annotations

import pytest
import torch

from minicpm_b200 import _lib, kv_pages
from test_gpu_kv_pages import KINDS, Pool, _caches, _layers

pytestmark = pytest.mark.gpu


def _recount(table, pool):
    refs = [0] * pool
    for row in table.tolist():
        for p in row:
            if p >= 0:
                refs[p] += 1
    return refs


def _reserve(pool, row, pages):
    """A scheduler's reservation: the row names pages before it has tokens."""
    pool.table[row][:len(pages)] = pages
    for p in pages:
        pool.refs[p] += 1


def _fork(pool, layers, state, parents, children):
    index = pool.dtype
    kv_pages.fork_sequences(layers, *state, torch.tensor(parents, dtype=index).cuda(),
                            torch.tensor(children, dtype=index).cuda())


@pytest.mark.parametrize("dtype,dim,hnd", KINDS[:2])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_a_childs_reserved_pages_are_given_back(dtype, dim, hnd, index):
    caches = _caches(2, 40, 16, 2, dim, dtype, seed=1, hnd=hnd)
    pool = Pool([100, 33, 16], 4, 16, 40, 9, caches, index, seed=3)
    free = [i for i in range(40) if pool.refs[i] == 0]
    _reserve(pool, 3, free[:9])  # every column
    _reserve(pool, 4, [free[9], pool.table[0][0]])  # one of them shared with row 0
    gpu, layers = _layers(caches, split=hnd)
    state = pool.gpu()
    _fork(pool, layers, state, [0, 1, 2], [3, 4, 5])
    pool.fork([0, 1, 2], [3, 4, 5])  # gives out pages by the counts before the call
    for p in [*free[:10], pool.table[0][0]]:
        pool.refs[p] -= 1
    pool.check(*state, gpu)
    assert pool.refs == _recount(state[0], 40)
    assert _lib.device_error() == _lib.DEVERR_NONE
    kv_pages.free_sequences(*state, torch.arange(7, device="cuda", dtype=index))
    assert state[2].abs().max().item() == 0 and (state[0] == -1).all()


def test_a_released_page_is_not_given_out_by_the_same_call():
    caches = _caches(1, 4, 16, 1, 64, torch.bfloat16)
    pool = Pool([20], 2, 16, 4, 3, caches)
    free = [i for i in range(4) if pool.refs[i] == 0]
    _reserve(pool, 1, free)
    gpu, layers = _layers(caches)
    state = pool.gpu()
    _fork(pool, layers, state, [0], [1])  # no page is free while the plan is made: not served, row 1 stays
    pool.check(*state, gpu)
    assert _lib.device_error() == _lib.DEVERR_NO_PAGE
    kv_pages.free_sequences(*state, torch.tensor([1], dtype=torch.int32).cuda())
    _fork(pool, layers, state, [0], [1])
    pool.free([1])
    pool.fork([0], [1])
    pool.check(*state, gpu)
    assert _lib.device_error() == _lib.DEVERR_NONE


def test_fork_into_the_row_of_a_bad_context():
    """keep leaves such a row with length 0 and its pages; so does a context of 0 with nothing accepted."""
    caches = _caches(1, 24, 16, 1, 64, torch.bfloat16, seed=2)
    pool = Pool([40, 50, 30], 0, 16, 24, 4, caches)
    _, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    acc, num = torch.tensor([[0, 1]] * 3, dtype=torch.int32).cuda(), torch.tensor([2, 2, 0], dtype=torch.int32).cuda()
    kv_pages.keep_accepted_tokens(layers, table, torch.tensor([-1, 48, 0], dtype=torch.int32).cuda(), acc, num, lens)
    assert lens.tolist() == [0, 50, 0] and _lib.device_error() == _lib.DEVERR_ACCEPT
    assert refs.tolist() == _recount(table, 24)
    _fork(pool, layers, (table, lens, refs), [1, 1], [0, 2])
    assert lens.tolist() == [50, 50, 50] and refs.tolist() == _recount(table, 24)
    assert sum(refs.tolist()) == 12 and max(refs.tolist()) == 3
    assert _lib.device_error() == _lib.DEVERR_NONE


def test_a_row_forked_from_itself_is_emptied():
    caches = _caches(1, 6, 16, 1, 64, torch.bfloat16)
    pool = Pool([20], 2, 16, 6, 3, caches)
    _reserve(pool, 1, [i for i in range(6) if pool.refs[i] == 0][:2])
    _, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    _fork(pool, layers, (table, lens, refs), [1], [1])  # its length is 0: a copy of an empty row
    assert table[1].tolist() == [-1, -1, -1] and lens.tolist() == [20, 0, 0]
    assert refs.tolist() == _recount(table, 6)
    assert _lib.device_error() == _lib.DEVERR_NONE


def test_bad_pages_of_a_child_row_are_recorded():
    caches = _caches(1, 8, 16, 1, 64, torch.bfloat16)
    pool = Pool([32], 2, 16, 8, 4, caches)
    _, layers = _layers(caches)
    table, lens, refs = pool.gpu()
    unused = int((refs == 0).nonzero()[0])
    for bad in (1 << 20, unused):  # past the pool; a page whose count is 0 already stays at 0
        table[1], lens[1] = -1, 0
        table[1, 3] = bad
        before = refs.clone()
        _fork(pool, layers, (table, lens, refs), [0], [1])
        assert lens.tolist() == [32, 32, 0] and table[1].tolist() == [*table[0, :2].tolist(), -1, -1]
        before[table[0, :2].long()] += 1
        assert torch.equal(refs, before)
        assert _lib.device_error() == _lib.DEVERR_PAGE_RANGE
