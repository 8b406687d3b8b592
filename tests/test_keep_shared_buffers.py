"""keep_accepted_tokens with the accepted paths in the buffer that the lengths are written to: other
warps read a path after the first of them has stored the sequence's length, so the call reads a copy."""

from __future__ import annotations

import pytest
import torch

from minicpm_b200 import _lib, kv_pages
from test_gpu_kv_pages import Pool, _caches, _keep_plain, _layers


class _Recorder:
    """The library with b200_keep_accepted replaced: notes the address of the paths that it is given."""

    def __init__(self, lib):
        self.lib, self.seen = lib, []

    def __getattr__(self, name):
        return getattr(self.lib, name)

    def b200_keep_accepted(self, caches, table, context, accepted, stride, most, counts, code, stream):
        self.seen.append((accepted, stride))
        return _lib.B200_OK


def _call(monkeypatch, acc, lens):
    """What the library would be given, on CPU tensors."""
    rec = _Recorder(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: rec)
    monkeypatch.setattr(_lib, "on_device", lambda dev: _lib._NO_SWITCH)
    monkeypatch.setattr(_lib, "current_stream", lambda dev: 0)
    monkeypatch.setattr(kv_pages, "_on", lambda layers, dev, what: None)
    n = lens.shape[0]
    kv_pages.keep_accepted_tokens(
        [torch.zeros(6, 2, 16, 2, 64)], torch.full((n, 4), -1, dtype=torch.int32), torch.zeros(n, dtype=lens.dtype), acc,
        torch.zeros(n, dtype=acc.dtype), lens)
    return rec.seen[0]


@pytest.mark.parametrize("at", [0, 1, 8, 9])
def test_paths_that_the_lengths_overwrite_are_read_from_a_copy(monkeypatch, at):
    state = torch.zeros(3, 4, dtype=torch.int32)
    lens = state.as_strided((3,), (1,), at)
    address, stride = _call(monkeypatch, state, lens)
    assert address != state.data_ptr() and stride == 4


def test_one_path_of_one_entry(monkeypatch):
    buf = torch.zeros(4, dtype=torch.int32)
    one = buf.as_strided((1, 1), (3, 2), 1)  # contiguous whatever its strides say
    assert _call(monkeypatch, one, buf[1:2])[0] != one.data_ptr()
    assert _call(monkeypatch, one, buf[2:3])[0] == one.data_ptr()


def test_paths_beside_the_lengths_are_read_in_place(monkeypatch):
    buf = torch.zeros(32, dtype=torch.int32)
    acc, lens = buf[3:15].view(3, 4), buf[:3]
    assert _call(monkeypatch, acc, lens) == (acc.data_ptr(), 4)
    assert _call(monkeypatch, buf[:12].view(3, 4), buf[12:15]) == (buf.data_ptr(), 4)
    wide = torch.zeros(3, 8, dtype=torch.int32)
    assert _call(monkeypatch, wide[:, :4], torch.zeros(3, dtype=torch.int32)) == (wide.data_ptr(), 8)


@pytest.mark.gpu
def test_lengths_in_the_paths_own_buffer():
    page, n = 16, 32
    caches = _caches(8, 200, page, 2, 128, torch.bfloat16, seed=3)
    pool = Pool([60] * n, 0, page, 200, 4, caches)
    gpu, layers = _layers(caches)
    table, _, refs = pool.gpu()
    ctx = [30 + i % 9 for i in range(n)]
    paths = [[i % 3, 4 + i % 2, 9, 17 - i % 4] for i in range(n)]
    state = torch.tensor(paths, dtype=torch.int32).cuda()
    lens = state.as_strided((n,), (1,), 7)
    kv_pages.keep_accepted_tokens(layers, table, torch.tensor(ctx, dtype=torch.int32).cuda(), state,
                                  torch.full((n,), 4, dtype=torch.int32).cuda(), lens)
    _keep_plain(caches, pool.table, ctx, paths, [4] * n, page)
    pool.lens = [c + 4 for c in ctx]
    pool.check(table, lens, refs, gpu)
    assert _lib.device_error() == _lib.DEVERR_NONE
