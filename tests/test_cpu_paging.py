"""Refusals of the block-table functions that need no GPU."""
from __future__ import annotations

import pytest
import torch

import hxlib


def test_entry_points_reject_bad_arguments_before_any_device_work():
    L = hxlib.lib()
    one = hxlib.ctypes.c_void_p(256)   # never read: every call below is refused on the host
    two = hxlib.ctypes.c_void_p(512)
    good = [None, one, 8, 1, 8, 16, one, one, one, 4, one, None, 4, two, two, two, two, 4, two, None]
    for i, bad in ((3, -1), (5, 0), (2, 7), (6, None), (13, None), (17, -1), (18, one), (14, one), (8, None), (12, -1)):
        args = list(good)
        args[i] = bad
        assert L.hx_tables_extend(*args) == hxlib.HX_ERR_ARG, i
    args = list(good)
    args[3] = 16385
    assert L.hx_tables_extend(*args) == hxlib.HX_ERR_UNSUPPORTED
    good = [None, one, 8, 1, 8, 16, one, one, one, 4, one, None, 4, two, two, None]
    for i, bad in ((3, -1), (5, 0), (2, 7), (6, None), (7, None), (10, None), (13, None), (14, None), (12, -1), (13, one),
                   (14, one)):
        args = list(good)
        args[i] = bad
        assert L.hx_tables_truncate(*args) == hxlib.HX_ERR_ARG, i
    assert L.hx_pool_reset_range(None, None, one, 1, one, one, None) == hxlib.HX_ERR_ARG


def test_cpu_tensors_are_refused():
    from kvquant import paging
    t = torch.zeros((2, 4), dtype=torch.int32)
    v = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(hxlib.HelixError):
        paging.extend_tables(t, v, v, v, v[:1], num_tokens=1)
    with pytest.raises(hxlib.HelixError):
        paging.truncate_tables(t, v, v, v, v[:1])
    with pytest.raises(ValueError):
        paging.extend_tables(v, v, v, v, v[:1], num_tokens=1)


def test_sizes_past_what_a_call_counts_are_refused():
    """A thread's token and page numbers stay in 32 bits up to 2^30 of them."""
    L = hxlib.lib()
    one, two = hxlib.ctypes.c_void_p(256), hxlib.ctypes.c_void_p(512)   # never read
    args = [None, one, 8, 1, 8, 16, one, one, one, 4, one, None, 4, two, two, two, two, (1 << 30) + 1, two, None]
    assert L.hx_tables_extend(*args) == hxlib.HX_ERR_UNSUPPORTED
    args[17] = 2 ** 31 - 1
    assert L.hx_tables_extend(*args) == hxlib.HX_ERR_UNSUPPORTED
