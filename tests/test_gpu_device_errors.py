"""Codes recorded by different kernels of the library (GPU): each is reported, none hides another."""

from __future__ import annotations

import pytest
import torch

from minicpm_b200 import _lib, kv_pages
from minicpm_b200.kv_cache import reshape_and_cache_flash

pytestmark = pytest.mark.gpu


def test_every_code_is_reported_once():
    assert _lib.device_error() == _lib.DEVERR_NONE
    cache = torch.zeros(4, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    rows = torch.ones(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    one = torch.ones(1, device="cuda")
    for _ in range(2):
        reshape_and_cache_flash(rows, rows, cache[:, 0], cache[:, 1], torch.tensor([4 * 16], device="cuda"), "auto", one, one)
        kv_pages.copy_pages([cache], torch.tensor([0], device="cuda"), torch.tensor([4], device="cuda"))
        assert {_lib.device_error(), _lib.device_error()} == {_lib.DEVERR_SLOT_RANGE, _lib.DEVERR_PAGE_RANGE}
        assert _lib.device_error() == _lib.DEVERR_NONE
    assert cache.abs().max().item() == 0.0
